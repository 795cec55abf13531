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
