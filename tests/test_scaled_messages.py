"""Refusals of the block-scaled operators say what they refuse, also where a workspace is asked for first."""
import pytest
import torch

import ctc_amd
from ctc_amd import _lib

EINVAL, EUNSUPPORTED = -1, -5


def refused(call):
    """(code, message) of a query, behind an unrelated error."""
    L = _lib.load()
    assert L.ctc_tc_get_option(b"no such option") < 0 and b"no such option" in L.ctc_tc_last_error()
    return call(L), L.ctc_tc_last_error().decode()


@pytest.mark.parametrize("args, code, text", [
    ((-1, 1, 1, 1), EINVAL, "negative size"), ((1, 1, 1, -5), EINVAL, "negative size"),
    ((1 << 31, 64, 64, 1), EUNSUPPORTED, "an extent is too large"), ((64, 64, 1 << 31, 1), EUNSUPPORTED, "an extent is too large"),
    ((64, 64, 64, 1 << 16), EUNSUPPORTED, "an extent is too large"),
])
def test_product_workspace_query(args, code, text):
    assert refused(lambda L: L.ctc_tc_scaled_workspace_bytes(*args)) == (code, "scaled_workspace_bytes: " + text)


@pytest.mark.parametrize("args, text", [
    ((-1, 2, 100), "negative size"), ((65, 2, 100), "at most 64 tokens"), ((4, 17, 100), "at most 16 experts a token"),
    ((4, 2, 1 << 31), "an extent is too large"),
])
def test_expert_workspace_query(args, text):
    code, message = refused(lambda L: L.ctc_tc_expert_workspace_bytes(*args))
    assert code == EINVAL and message.startswith("expert_workspace_bytes: " + text)


@pytest.mark.gpu
def test_python_calls_pass_on_what_the_operator_refuses(cuda):
    codes = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)  # noqa: E731
    ones = lambda *shape: torch.ones(shape, device=cuda)  # noqa: E731

    def layer(tokens, top):
        x = torch.zeros(tokens, 128, dtype=torch.bfloat16, device=cuda)
        pick = torch.zeros(tokens, top, dtype=torch.int32, device=cuda)
        return ctc_amd.expert_layer(x, codes(2, 256, 128), ones(2, 2, 1), codes(2, 128, 128), ones(2, 1, 1), pick, ones(tokens, top))

    def product(batch):
        return ctc_amd.scaled_contract(codes(batch, 33, 16), ones(batch, 33, 1), codes(1, 1, 16).expand(batch, 1, 16), ones(1, 1, 1).expand(batch, 1, 1))

    for call, text in ((lambda: layer(65, 2), "expert_layer: at most 64 tokens"), (lambda: layer(4, 17), "expert_layer: at most 16 experts a token"),
                       (lambda: product(1 << 16), "scaled_contract: an extent is too large")):
        assert _lib.load().ctc_tc_get_option(b"no such option") < 0
        with pytest.raises(ctc_amd.CtcError, match=text) as caught:
            call()
        assert caught.value.code == EUNSUPPORTED
