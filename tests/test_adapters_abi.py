"""CPU tests of the adapters' and heads' entry points: without a context they answer with a status, whatever else they get."""
import pytest

import lib_b200
from lib_b200 import _capi

CALLS = {"qm_lora_create": (8, 32, 1, 1, 1, None), "qm_lora_destroy": (None,), "qm_lora_set": (None, 0, 1, 1.0, 0, 0, 0),
         "qm_lora_matvec": (None, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0), "qm_lora_matmul_bf16": (None, 0, 1, 0, 0, 0, 0, 0, 0),
         "qm_lora_backward": (None, 0, 0, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0), "qm_matvec_lora": (0, None, 0, 0, 1, 0, 0, 0, 0, 0),
         "qm_matmul_bf16_lora": (0, None, 0, 1, 0, 0, 0, 0), "qm_rope_create": (8, 8, 1.0, None, 0, None), "qm_rope_destroy": (None,),
         "qm_qk_norm_rope": (None, 0, 0, 1, 1, 1, 0, 0, 0.0, 0, 0, 0, 0, 0, 0),
         "qm_qk_norm_rope_backward": (None, 0, 0, 1, 1, 1, 0, 0, 0.0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)}


@pytest.mark.parametrize("name", CALLS)
def test_no_context(name):
    assert name in _capi.declared_symbols()
    assert getattr(lib_b200.lib, name)(None, *CALLS[name]) == -5
