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
