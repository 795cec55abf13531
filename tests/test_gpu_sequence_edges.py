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


# ---------------------------------------------------------------------------------------------
# linear attention against float64, value by value
# ---------------------------------------------------------------------------------------------
def la_exact(s, scale=None):
    """{name: (value, the same sum with every term's magnitude)} of out, state, dq, dk, dv, d_state."""
    sc = s["q"].shape[3] ** -0.5 if scale is None else scale

    def run(f, sc):
        ls = [f(s[n].double()).requires_grad_() for n in ("q", "k", "v", "state") if s[n] is not None]
        out, last = la_plain(*ls[:3], s["ld"].double(), sc, ls[3] if len(ls) > 3 else None, s["reset"], s["lengths"])
        gr = torch.autograd.grad([out, last], ls, [f(s["d_out"].double()), f(s["d_state"].double())], allow_unused=True)
        return [out.detach(), last.detach()] + [torch.zeros_like(x) if g is None else g for g, x in zip(gr, ls)]
    return dict(zip(("out", "state", "dq", "dk", "dv", "d_state"), zip(run(lambda x: x, sc), run(torch.abs, abs(sc)))))


def la_close(exact, got, s, dtype):
    """Every value a number, off by at most the additions of its float32 sum and its own rounding: the dot
    products over D, the walk over T, head groups, and the decays lam^n (up to 40 u where it still counts)."""
    n = (s["q"].shape[3] + s["v"].shape[3] + s["q"].shape[1] + 16 + 64) * U
    for name, a in got.items():
        (b, m), a = exact[name], a.detach().cpu().double()
        assert a.shape == b.shape, name
        tol = n * m + (0 if "state" in name else torch.finfo(dtype).eps / 2 * b.abs() + (2.0 ** -25 if dtype == F16 else 0))
        ok = (a - b).abs() <= tol + 1e-300
        assert ok.all(), f"{name}: {int((~ok).sum())} of {ok.numel()} off, {int(torch.isnan(a).sum())} NaN"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T, heads", [(70, (2, 2, 2)), (70, (1, 2, 1)), (700, (2, 2, 2)), (700, (1, 1, 2))])
def test_la_only_the_wanted_gradients(K, dtype, T, heads):
    """Each subset of the gradients is right by itself, and nothing is computed or stored for the others."""
    s = la_inputs(2, T, 2, heads, 40, 24, dtype, seed=T, reset=0.01, lengths=[T, T // 2 + 3])
    exact = la_exact(s)
    names = ("q", "k", "v", "state")
    dev = {n: s[n].cuda() for n in names}
    ld, rs, ln = (s[n].cuda() for n in ("ld", "reset", "lengths"))
    raw = K.linear_attention_backward
    for some in range(1, 16):
        on = [bool(some >> i & 1) for i in range(4)]
        x = {n: t.clone().requires_grad_(w) for (n, t), w in zip(dev.items(), on)}
        out, last = K.linear_attention(x["q"], x["k"], x["v"], ld, state=x["state"], reset=rs, lengths=ln, return_state=True)
        made = []
        with pytest.MonkeyPatch.context() as mp:
            mp.setattr(K, "linear_attention_backward", lambda *a, **k: made.append(raw(*a, **k)) or made[-1])
            got = torch.autograd.grad([out, last], [t for t in x.values() if t.requires_grad],
                                      [s["d_out"].cuda(), s["d_state"].cuda()])
        assert [g is not None for g in made[0]] == on
        la_close(exact, dict(zip([("d_state" if n == "state" else "d" + n) for n, w in zip(names, on) if w], got)), s, dtype)


def test_la_raw_backward_without_any_gradient(K):
    s = la_inputs(1, 5, 1, (1, 1, 1), 4, 4, F32, seed=1)
    args = [s[n].cuda() for n in ("q", "k", "v", "ld")]
    res = K.linear_attention_backward(s["d_out"].cuda(), None, *args, state=s["state"].cuda(), want=(False,) * 4)
    assert res == (None,) * 4


def la_run(K, s, scale=None):
    """{name: value} of out, state and all gradients."""
    x = {n: s[n].cuda().requires_grad_() for n in ("q", "k", "v", "state") if s[n] is not None}
    opt = {n: s[n].cuda() for n in ("reset", "lengths") if s[n] is not None}
    out, last = K.linear_attention(x["q"], x["k"], x["v"], s["ld"].cuda(), scale=scale, state=x.get("state"),
                                   return_state=True, **opt)
    got = torch.autograd.grad([out, last], list(x.values()), [s["d_out"].cuda(), s["d_state"].cuda()])
    return dict(out=out, state=last, **{"d_state" if n == "state" else "d" + n: g for n, g in zip(x, got)})


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, T, H, heads, Dk, Dv", [
    (1, 1, 1, (1, 1, 1), 1, 1), (2, 31, 2, (2, 2, 2), 5, 7), (1, 32, 3, (3, 3, 3), 32, 32),
    (3, 33, 2, (2, 2, 2), 33, 65), (2, 64, 4, (1, 2, 4), 64, 64), (1, 65, 4, (4, 2, 1), 64, 128),
    (1, 129, 2, (2, 2, 2), 128, 128), (2, 97, 6, (3, 2, 6), 128, 40), (1, 130, 2, (1, 1, 2), 96, 100),
    (1, 511, 2, (2, 1, 2), 17, 128)])
def test_la_values_of_all_shapes(K, dtype, B, T, H, heads, Dk, Dv):
    for more in (dict(), dict(reset=0.03, time_major=True), dict(state=False, lengths=[max(0, T - 9 * b) for b in range(B)])):
        s = la_inputs(B, T, H, heads, Dk, Dv, dtype, seed=T + Dv, **more)
        la_close(la_exact(s), la_run(K, s), s, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T, D", [(512, 16), (700, 64), (1281, 128)])
def test_la_values_of_split_sequences(K, dtype, T, D):
    s = la_inputs(1, T, 2, (1, 2, 2), D, D, dtype, seed=T, reset=0.004)
    s["reset"][0, 256] = 1
    la_close(la_exact(s), la_run(K, s), s, dtype)
    s["reset"], s["lengths"] = None, torch.tensor([T - 200], dtype=torch.int32)
    la_close(la_exact(s), la_run(K, s), s, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 128])
def test_la_values_of_all_decays(K, dtype, D):
    s = la_inputs(2, 150, 4, (4, 4, 4), D, D, dtype, seed=3, reset=0.02)
    s["ld"] = torch.tensor([float("-inf"), -20.0, 0.0, -0.5])
    la_close(la_exact(s, scale=-1.5), la_run(K, s, scale=-1.5), s, dtype)
    la_close(la_exact(s), la_run(K, s), s, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, H, T, Dk, Dv", [(260, 8, 100, 7, 9), (256, 8, 97, 12, 33), (130, 16, 70, 33, 20),
                                            (64, 33, 65, 5, 50), (256, 8, 66, 70, 5)])
def test_la_many_short_sequences(K, dtype, B, H, T, Dk, Dv):
    """Blocks enough, of up to 64 columns: 32 tokens a chunk on bf16, several chunks a sequence."""
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, T + 1, (B,), generator=g)
    lengths[:6] = torch.tensor([T, 32, 33, 64, 0, 1])
    s = la_inputs(B, T, H, (H, H, H), Dk, Dv, dtype, seed=B, reset=0.02, lengths=lengths.tolist())
    s["reset"][0, 31] = s["reset"][0, 32] = s["reset"][1, 31] = s["reset"][3, 32] = s["reset"][3, 63] = s["reset"][6, 64] = 1
    la_close(la_exact(s), la_run(K, s), s, dtype)


# ---------------------------------------------------------------------------------------------
# infs and NaNs: what they do not reach keeps its digits
# ---------------------------------------------------------------------------------------------
def keep_close(exact, got, s, dtype, keep):
    """la_close of the values of keep[name]."""
    pick = {n: (exact[n][0][k], exact[n][1][k]) for n, k in keep.items()}
    la_close(pick, {n: got[n].detach().cpu()[k] for n, k in keep.items()}, s, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("B, H, T, D, at", [(2, 2, 200, 64, 42), (2, 2, 200, 128, 63), (2, 2, 130, 20, 31), (260, 8, 100, 10, 32),
                                            (260, 8, 100, 10, 45), (1, 2, 700, 32, 300)])
def test_la_other_episodes_keep_their_digits(K, dtype, bad, B, H, T, D, at):
    """A spoilt token in an episode of ten: all other episodes' outputs and gradients as if it were not there."""
    s = la_inputs(B, T, H, (H, 1, H), D, D, dtype, seed=at, reset=1e-9)
    first, last = at - 3, at + 7
    s["reset"][:, first] = s["reset"][:, last] = s["reset"][:, T - 9] = 1
    clean = dict(s)
    for n in ("q", "k", "v", "d_out"):
        clean[n] = s[n].clone()
        clean[n][0, first:last] = 0
        s[n][0, at, 0, 3] = bad
    exact, got = la_exact(clean), la_run(K, s)
    rows = torch.ones(B, T, dtype=torch.bool)
    rows[0, first:last] = False
    keep = {n: rows for n in ("out", "dq", "dk", "dv")}
    keep_close(exact, got, s, dtype, {**keep, "state": slice(None), "d_state": slice(None)})
    assert not torch.isfinite(got["out"][0, at:last]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [[0], [31], [32], [33, 34], [63, 64], [20, 22, 130], [149]])
def test_la_other_tokens_keep_their_digits(K, dtype, bad, at):
    """A spoilt value reaches its own column from its token on, a spoilt d_out the gradients up to its token."""
    s = la_inputs(2, 150, 2, (2, 2, 2), 33, 40, dtype, seed=15)
    clean = {n: (x.clone() if torch.is_tensor(x) else x) for n, x in s.items()}
    out_ok = torch.ones(2, 150, 2, 40, dtype=torch.bool)
    for i, t in enumerate(at):
        s["v"][0, t, 0, 5 + i], clean["v"][0, t, 0, 5 + i] = bad, 0
        out_ok[0, t:, 0, 5 + i] = False
    exact = la_exact(clean)
    out, last = K.linear_attention(*(s[n].cuda() for n in "qkv"), s["ld"].cuda(), state=s["state"].cuda(), return_state=True)
    assert torch.equal(torch.isfinite(out.cpu()), out_ok)
    keep_close(exact, dict(out=out, state=last), s, dtype, dict(out=out_ok, state=out_ok[:, -1].unsqueeze(2).expand(2, 2, 33, 40)))
    # backward
    s = la_inputs(2, 150, 2, (2, 2, 2), 33, 40, dtype, seed=15)
    clean = {n: (x.clone() if torch.is_tensor(x) else x) for n, x in s.items()}
    dk_ok, dv_ok, dq_ok = (torch.ones(2, 150, 2, n, dtype=torch.bool) for n in (33, 40, 33))
    for i, t in enumerate(at):
        s["d_out"][0, t, 1, 5 + i], clean["d_out"][0, t, 1, 5 + i] = bad, 0
        dk_ok[0, :t + 1, 1] = dq_ok[0, t, 1] = False
        dv_ok[0, :t + 1, 1, 5 + i] = False
    got = la_run(K, s)
    keep_close(la_exact(clean), got, s, dtype, dict(dq=dq_ok, dk=dk_ok, dv=dv_ok))
    assert not torch.isfinite(got["dk"].cpu()[~dk_ok]).all()


# ---------------------------------------------------------------------------------------------
# one token: states beyond the last-level cache
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B, H, Dk, Dv", [(4300, 4, 64, 61), (8500, 4, 64, 31), (2200, 4, 128, 62), (600, 4, 120, 128)])
def test_la_step_past_the_caches(K, dtype, B, H, Dk, Dv):
    """The same envs in a small call have the same bits, and those are within a few roundings of float64."""
    g = torch.Generator(device="cuda").manual_seed(B)
    apart = B * H * Dk * Dv * 4 <= 256 << 20             # only read and written states together are beyond it
    q, k = (torch.randn(B, H, Dk, device="cuda", generator=g).to(dtype) for _ in range(2))
    v = torch.randn(B, H, Dv, device="cuda", generator=g).to(dtype)
    ld = -torch.rand(H, device="cuda", generator=g)
    st = torch.randn(B, H, Dk, Dv, device="cuda", generator=g)
    rs = torch.rand(B, device="cuda", generator=g) < 0.3
    st[rs.nonzero()[0]] = float("nan")                   # dropped
    few = torch.cat([torch.arange(100), torch.arange(B - 100, B)]).cuda()
    small = st[few].clone()
    old = torch.where(rs[few].view(-1, 1, 1, 1), 0.0, small).cpu().double()
    o1 = K.linear_attention_step(q[few], k[few], v[few], ld, small, reset=rs[few])
    new = torch.full_like(st, 7.0)
    o2 = K.linear_attention_step(q, k, v, ld, st, reset=rs, state_out=new)
    assert torch.equal(o2[few], o1) and torch.equal(new[few], small)
    if not apart:
        o3 = K.linear_attention_step(q, k, v, ld, st, reset=rs)
        assert torch.equal(o3, o2) and torch.equal(st, new)
    c = [t[few].cpu().double() for t in (q, k, v)]
    lam = torch.exp(ld.cpu().double()).view(1, H, 1, 1)
    want = lam * old + c[1].unsqueeze(-1) * c[2].unsqueeze(-2)
    mag = lam * old.abs() + c[1].abs().unsqueeze(-1) * c[2].abs().unsqueeze(-2)
    assert ((small.cpu().double() - want).abs() <= 8 * U * mag).all()
    out, om = ((f(c[0]).unsqueeze(-1) * m).sum(-2) * Dk ** -0.5 for f, m in ((lambda x: x, want), (torch.abs, mag)))
    assert ((o1.cpu().double() - out).abs() <= torch.finfo(dtype).eps / 2 * out.abs() + (Dk + 16) * U * om).all()


# ---------------------------------------------------------------------------------------------
# token log-probabilities: rows both split and past the caches, rows of 64 parts
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, N, V, part", [(BF16, 300, 900001, 225280), (F32, 150, 900003, 129024)])
@pytest.mark.parametrize("k", [0, 5])
def test_lp_split_rows_past_the_caches(K, dtype, N, V, part, k):
    """Fewer than 512 rows of more than 512 MB together: parts of rows, each from a multiple of 16 bytes on."""
    g = torch.Generator(device="cuda").manual_seed(V)
    flat = torch.empty(N * V + 1, dtype=dtype, device="cuda").normal_(0.0, 3.0, generator=g)
    x = flat[1:].view(N, V)
    x[9], x[9, V - 1] = float("-inf"), 0.5
    x[10, :V // 2] = float("-inf")
    x[11] = torch.finfo(dtype).min
    x[12, part - 10:part + 3] = 20.0                           # ties over a part's border
    x[13, part - 6:part + 5] = 20.0
    pick = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, N - 1])
    tokens = torch.randint(0, V, (N,), device="cuda", generator=g)
    tokens[5], tokens[9] = -1, V - 1
    res = K.token_logprob(x, tokens, top_k=k)
    rows, tk = x[pick.cuda()].cpu(), tokens[pick.cuda()].cpu()
    r = lp_plain(rows, tk, 1.0, k)
    base = (V / 64 + 48 + 6 * torch.nan_to_num(r["spread"])) * U
    fin = lambda t: torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t))

    def close(a, b, tol):
        a = a[pick.cuda()].cpu().double()
        assert (((a - b).abs() <= tol) | (a == b)).all()
    close(res[0], r["logp"], base + 6 * U * fin(r["logp"]))
    close(res[1], r["entropy"], base * (2 + 2 * r["spread"]))
    if k:
        assert torch.equal(res[3][pick.cuda()].cpu(), r["top_tokens"])
        close(res[2], r["top_logp"], base[:, None] + 6 * U * fin(r["top_logp"]))


@pytest.mark.parametrize("dtype, V", [(BF16, 262000), (F32, 131000)])
@pytest.mark.parametrize("k", [0, 1, 32])
def test_lp_rows_of_64_parts(K, dtype, V, k):
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(7, V, generator=g) * 3).to(dtype)
    logits[1] = torch.randint(0, 3, (V,), generator=g).to(dtype)
    logits[2, :-40] = float("-inf")
    logits[3], logits[3, V // 2] = float("-inf"), 1.0
    logits[4] = torch.arange(V).to(dtype) * 1e-4
    tokens = torch.randint(0, V, (7,), generator=g)
    tokens[6] = -1
    lp_check(K, logits, tokens, k=k)


@pytest.mark.parametrize("dtype, bits", [(F32, 0x7F800001), (BF16, 0x7F81), (F16, 0x7C01)])
@pytest.mark.parametrize("V", [9, 100, 200, 300, 3000, 20000])
@pytest.mark.parametrize("k", [1, 2, 5])
def test_lp_alternatives_beside_nans_of_any_kind(K, dtype, bits, V, k):
    """NaNs of either sign, quiet and signalling, beside the best logits: no alternatives, and none is lost."""
    g = torch.Generator().manual_seed(V + k)
    N = 600                                               # rows enough that none is split
    logits = torch.randn(N, V, generator=g).to(dtype)
    best = torch.randint(0, V - 1, (N,), generator=g)
    logits[torch.arange(N), best] = 50.0
    raw = logits.view(torch.int32 if dtype == F32 else torch.int16)
    low = torch.iinfo(raw.dtype).min
    for i in range(N):
        at = int(best[i]) + 1 if i % 3 else int(torch.randint(0, V, (1,), generator=g))
        at = at if at != int(best[i]) else at + 1
        raw[i, at] = bits + (low if i % 2 else 0) + (torch.finfo(dtype).bits == 32 and i % 5 == 0) * 0x400000
        if i % 4 == 0:                                    # a whole lane's vector, and the next one
            raw[i, max(0, at - 5):at] = torch.where(logits[i, max(0, at - 5):at] == 50.0, raw[i, max(0, at - 5):at],
                                                    torch.tensor(bits, dtype=raw.dtype))
    assert torch.isnan(logits).any(-1).all()
    want = lp_plain(logits, torch.zeros(N, dtype=torch.int64), 1.0, k)["top_tokens"]
    for n in (N, 9):                                      # 9 long rows: in parts
        logp, ent, tl, tt = K.token_logprob(logits[:n].cuda(), torch.zeros(n, dtype=torch.int64, device="cuda"), top_k=k)
        assert torch.isnan(logp).all() and torch.isnan(ent).all() and torch.isnan(tl).all()
        some = (~torch.isnan(logits[:n])).sum(-1, keepdim=True) > torch.arange(k)   # as many numbers as that
        assert torch.equal(tt.cpu(), torch.where(some, want[:n], -1))


def test_sequence_operators_in_inference_mode(K):
    s = la_inputs(2, 40, 2, (2, 2, 2), 16, 16, F32, seed=3)
    q, k, v, ld, st = (s[n].cuda() for n in ("q", "k", "v", "ld", "state"))
    logits, tokens = torch.randn(3, 700, device="cuda"), torch.arange(3, device="cuda")
    want = K.linear_attention(q, k, v, ld, state=st, return_state=True) + K.token_logprob(logits, tokens, top_k=2)
    step = K.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st.clone())
    with torch.inference_mode():
        got = K.linear_attention(q, k, v, ld, state=st, return_state=True) + K.token_logprob(logits, tokens, top_k=2)
        mem = st.clone()
        assert torch.equal(K.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, mem), step)
        assert not torch.equal(mem, st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
