"""The sequence-policy operators where they can go wrong unseen: outputs that are small beside their terms,
comparisons that a NaN cannot pass, and the kernels' variants that only large calls reach. Against the plain
restatements in float64 of test_gpu_sequence.py; tolerances count roundings (u = 2^-24) as there."""
import math

import pytest
import torch

from test_gpu_sequence import BF16, F16, F32, U, K, la_inputs, la_plain, lp_check, lp_plain  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# outputs that are small beside their terms
# ---------------------------------------------------------------------------------------------
FINE = 1.0 + 2.0 ** -10 + 2.0 ** -19   # three bfloat16 numbers; two hold it to 2^-19


@pytest.mark.parametrize("D", [8, 32, 64, 128])
@pytest.mark.parametrize("T", [20, 130])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_la_pairs_cancel(K, dtype, T, D):
    """q k of FINE and 1 + 2^-10 with opposite values: what is left is 2^-19 of the terms. Every product and
    partial sum is a multiple of 2^-19 below 4, so a float32 sum has it exactly in any order; T = 130 also
    takes it through the state."""
    q = torch.zeros(1, T, 1, D)
    k, v = torch.zeros_like(q), torch.zeros_like(q)
    q[..., :3] = 1.0
    k[0, 3, 0, :3] = torch.tensor([1.0, 2.0 ** -10, 2.0 ** -19])
    k[0, 4, 0, :2] = torch.tensor([1.0, 2.0 ** -10])
    x = torch.tensor([1.0, -1.0, 2.0, 0.5]).repeat(D // 4)
    v[0, 3, 0], v[0, 4, 0] = x, -x
    out = K.linear_attention(*(t.to(dtype).cuda() for t in (q, k, v)), torch.zeros(1, device="cuda"), scale=1.0)
    assert torch.equal(out[0, 4:, 0].float().cpu(), (2.0 ** -19 * x).expand(T - 4, D))


@pytest.mark.parametrize("D", [8, 32, 64, 128])
@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_la_state_cancels(K, dtype, T, D):
    """The same of two rows of the state that comes in."""
    x = torch.tensor([1.0, -1.0, 2.0, 0.5]).repeat(D // 4)
    state = torch.zeros(1, 1, D, D)
    state[0, 0, 0], state[0, 0, 1] = FINE * x, -(1.0 + 2.0 ** -10) * x
    q = torch.zeros(1, T, 1, D, dtype=dtype, device="cuda")
    z = torch.zeros_like(q)
    q[..., :2] = 1.0
    out = K.linear_attention(q, z, z, torch.zeros(1, device="cuda"), scale=1.0, state=state.cuda())
    assert torch.equal(out[0, :, 0].float().cpu(), (2.0 ** -19 * x).expand(T, D))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_la_weighted_values_cancel(K, dtype, D):
    """dv of a token two chunks before two others: FINE (do_a + 0.75 do_b) with do_b about -do_a / 0.75. The
    weighted values, their two additions to the state, its product with k and the next chunk's decay of 1
    are a rounding each: 8 u of the terms at most."""
    g = torch.Generator().manual_seed(D)
    T = 140
    q, k, v, do = (torch.zeros(1, T, 1, D) for _ in range(4))
    k[0, 0, 0, 0] = 1.0
    q[0, 130, 0, 0], q[0, 131, 0, 0] = 1.0, 0.75
    do[0, 130] = torch.randn(D, generator=g).to(BF16).float()
    do[0, 131] = (-do[0, 130] / 0.75).to(BF16).float()
    ins = [t.to(dtype).cuda().requires_grad_() for t in (q, k, v)]
    out = K.linear_attention(*ins, torch.zeros(1, device="cuda"), scale=FINE)
    dv = torch.autograd.grad(out, ins, do.to(dtype).cuda())[2][0, 0, 0].cpu().double()
    a, b = do[0, 130, 0].double(), 0.75 * do[0, 131, 0].double()
    want = FINE * (a + b)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 8 * U * FINE * (a.abs() + b.abs())
    assert ((dv - want).abs() <= tol).all()


# ---------------------------------------------------------------------------------------------
# empty batches
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("V", [7, 512, 513, 40000])
def test_lp_no_rows(K, V):
    x = torch.zeros(0, V, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    logp, ent, tl, tt = K.token_logprob(x, t, top_k=2)
    assert logp.shape == ent.shape == (0,) and tl.shape == tt.shape == (0, 2)
    assert torch.autograd.grad(logp.sum() + ent.sum(), [x])[0].shape == (0, V)
    logp, ent = K.token_logprob(x.detach().view(3, 0, V), t.view(3, 0))
    assert logp.shape == ent.shape == (3, 0)


# ---------------------------------------------------------------------------------------------
# token log-probabilities: maxima that rise through |m log2(e) / temperature| = 1e6, where the exponents'
# form changes
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("temperature", [1.0, 1e-3, 0.37])
@pytest.mark.parametrize("V", [513, 3000, 20000])
def test_lp_rising_through_the_border(K, V, temperature, sign):
    """Values of neighbouring logits on either side, the larger ones behind, so that each lane's sums move
    from one form to the other; a few steps apart, so that the sums before count in the result."""
    g = torch.Generator().manual_seed(V)
    border = 1e6 / 1.4426950408889634 * temperature
    step = max(math.ulp(border) * 2.0 ** 29, 0.25 * temperature)   # a float32 step, or a quarter of the temperature
    N = 520                              # rows enough that none is split, so a wave takes tile after tile
    at = torch.linspace(-6.0, 6.0, V).expand(N, V) + 0.3 * torch.randn(N, V, generator=g)
    at[1::8] = -at[1::8]                              # falling
    at[2::8, :-1], at[2::8, -1] = -2.0, 2.0           # one step at the end
    at[3::8] = at[3::8].abs() - 1.0
    at[4::8] = torch.where(torch.arange(V) % 1024 < 512, -2.0, 2.0)
    logits = (sign * border + at.double() * step).float()
    lp_check(K, logits, torch.randint(0, V, (N,), generator=g), temperature=temperature, k=5)
