"""What the backward of packed attention asks for as workspace, and refusals that
take sizes of their own: made on the host, before any launch (no GPU)."""

import pytest

from test_library import raw  # noqa: F401  (the fixture)
from test_packed_abi import BF16, EINVAL, EWORKSPACE, F16, F32, backward, gradient, lib, logprobs, th  # noqa: F401

TERMS = 2 * 4  # bytes a row and query head: two floats


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,h,hk,d,split", [
    (100, 4, 2, 64, True), (16384, 32, 8, 128, False), (65536, 32, 8, 128, False), (16384, 12, 12, 64, None),
    # the last sizes of fewer than 512 tiles of keys and K/V heads, of 128 rows up to 192 channels and of 64 above, and the first past them
    (128 * 64 - 1, 16, 8, 192, False), (128 * 63 - 1, 16, 8, 192, True), (64 * 64 - 1, 16, 8, 200, False), (64 * 63 - 1, 16, 8, 200, True),
])
def test_backward_workspace(lib, dtype, tokens, h, hk, d, split):  # noqa: F811
    """Two floats a query row, and f32 partials of dK and dV only where a call takes them."""
    layout = 64 if d <= 64 else 128 if d <= 128 else 256
    terms, parts = TERMS * h * tokens + 512, 2 * 4 * h * tokens * layout
    most = lib.mi355x_packed_attn_bwd_workspace_bytes(3, tokens, h, hk, d)
    need = lib.mi355x_packed_attn_bwd_workspace_bytes_for(3, tokens, h, hk, d, dtype)
    assert most == (terms if hk == h else terms + parts)
    assert need == (most if dtype == F32 or split else terms)
    s = th(h * d, d)
    over = dict(tokens=tokens, heads=h, kv_heads=hk, d=d, dtype=dtype, **dict.fromkeys(("dqt", "dkt", "dvt", "dot", "qt", "kt", "vt", "ot"), s))
    assert backward(lib, wsb=need - 1, **over) == EWORKSPACE


def test_logprobs_of_the_largest_vocabularies(lib):  # noqa: F811
    """A row's walk counts elements in 32 bits, up to a batch past its end."""
    most = 2 ** 31 - 2 ** 14
    for c in (most, 2 ** 31 - 1):
        assert logprobs(lib, n=600, c=c, ld=0, top=0, tt=None, tlp=None) == EINVAL
        assert gradient(lib, n=600, c=c, ld=0, ld_dx=c, top=0) == EINVAL
        assert lib.mi355x_token_logprobs_workspace_bytes(600, c, 0, BF16) == -1
    assert lib.mi355x_token_logprobs_workspace_bytes(600, most - 1, 0, BF16) == 0
