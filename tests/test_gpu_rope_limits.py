"""More tokens than the heads' kernels count are refused before anything is launched."""
import pytest

import lib_b200
from lib_b200 import _capi

pytestmark = pytest.mark.gpu

LIMIT = -11


def test_token_limit(ctx):
    rope = ctx.rope(8, 8, 10000.0)
    for tokens in ((1 << 30) + 1, (1 << 31) - 1):      # (without memory: refused for that where the limit is not looked at)
        for call in (lambda: rope.qk_norm(0, 8, tokens, 1, 0, 0, 0, 0.0, 0, 0, 8, 0, 0),
                     lambda: rope.qk_norm_backward(0, 8, tokens, 1, 0, 0, 0, 0.0, 0, 0, 8, 0, 0, 0, 8, 0, 0, _capi.QK_NO_NORM)):
            with pytest.raises(lib_b200.QmError) as e:
                call()
            assert e.value.code == LIMIT
    rope.close()
