"""Calls of the sequence-policy operators (linear attention, token log-probabilities) that are answered or
refused on the host, before any launch."""
import ctypes as C

import pytest
import torch

from reinforcementlearningplatform_amd import _abi, _native
from reinforcementlearningplatform_amd import kernels as K  # noqa: F401
from reinforcementlearningplatform_amd._native import RLPError  # noqa: F401

DEV = C.c_void_p(1 << 20)  # never dereferenced: nothing is launched


@pytest.mark.parametrize("vocab", [1, 512, 513, 50257, 0x7FF00000])
@pytest.mark.parametrize("top_k", [0, 1])
def test_token_logprob_without_rows(vocab, top_k):
    """An empty batch needs no scratch and launches nothing, whatever its rows' length."""
    lib = _native.lib()
    for dtype in (_abi.RLP_F32, _abi.RLP_BF16):
        assert lib.rlp_token_logprob_workspace_bytes(0, vocab, top_k, dtype) == 0
        assert lib.rlp_token_logprob(DEV, dtype, 0, vocab, vocab, DEV, 1.0, top_k, DEV, DEV, DEV, DEV, DEV, None, 0,
                                     None) == 0
        assert lib.rlp_token_logprob_backward(DEV, dtype, 0, vocab, vocab, DEV, 1.0, DEV, DEV, DEV, DEV, vocab,
                                              None) == 0


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """A tangent does not show in requires_grad; the operators raise instead of returning none."""
    import torch.autograd.forward_ad as fwd
    q, k, v = (torch.ones(2, 3, 2, 4) for _ in range(3))
    ld, state = -torch.ones(2), torch.ones(2, 2, 4, 4)
    logits, tokens = torch.ones(3, 5), torch.zeros(3, dtype=torch.int64)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        def dual(x):
            return fwd.make_dual(x, torch.ones_like(x))
        args = dict(q=q, k=k, v=v, log_decay=ld, state=state)
        for name in args:
            with pytest.raises(RLPError, match="forward-mode"):
                K.linear_attention(**{**args, name: dual(args[name])})
        step = dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], log_decay=ld, state=state, state_out=state.clone(),
                    out=torch.ones(2, 2, 4))
        for name in step:
            with pytest.raises(RLPError, match="forward-mode"):
                K.linear_attention_step(**{**step, name: dual(step[name])})
        with pytest.raises(RLPError, match="forward-mode"):
            K.token_logprob(dual(logits), tokens)
        # no tangent: on to the next check, of the device
        for call in (lambda: K.linear_attention(**args), lambda: K.linear_attention_step(**step),
                     lambda: K.token_logprob(logits, tokens)):
            with pytest.raises(RLPError, match="GPU"):
                call()
    with pytest.raises(RLPError, match="forward-mode"):
        torch.func.jvp(lambda x: K.token_logprob(x, tokens)[0], (logits,), (logits,))


def step_call(**over):
    """rlp_linear_attention_step on made-up addresses, 1 MB apart: 2 x 4 heads, 16 x 16, float32."""
    c = _abi.LACfg()
    for name, x in dict(dtype=0, B=2, T=1, H=4, Hq=4, Hk=4, Hv=4, Dk=16, Dv=16, scale=1.0).items():
        setattr(c, name, x)
    for name in ("q_stride", "k_stride", "v_stride", "o_stride"):
        setattr(c, name, (C.c_int64 * 3)(64, 0, 16))
    c.reset_stride = (C.c_int64 * 2)(1, 0)
    names = ("q", "k", "v", "log_decay", "reset", "state", "state_out", "out")
    at = {n: (i + 1) << 20 for i, n in enumerate(names)}
    at["state_out"] = at["state"]
    at.update(over)
    rc = _native.lib().rlp_linear_attention_step(C.byref(c), *(C.c_void_p(at[n]) for n in names), None)
    return rc, _native.lib().rlp_last_error_string()


STATE = 6 << 20   # 8192 bytes of states, 512 of the outputs, q, k and v, 16 of log_decay, 2 of reset


@pytest.mark.parametrize("over, word", [
    (dict(q=STATE), b"updated state"), (dict(k=STATE + 8191), b"updated state"), (dict(v=STATE - 511), b"updated state"),
    (dict(log_decay=STATE + 100), b"updated state"), (dict(reset=STATE - 1), b"updated state"),
    (dict(out=STATE + 8188), b"out overlaps"), (dict(out=STATE - 511), b"out overlaps"),
    (dict(state_out=STATE + 4), b"state_out overlaps"), (dict(state_out=STATE - 8188), b"state_out overlaps")])
def test_step_refuses_what_it_would_overwrite(over, word):
    """The state that is updated in place is written as well as out: blocks of other heads still read the rest."""
    rc, message = step_call(**over)
    assert rc == _abi.RLP_EINVAL and word in message
