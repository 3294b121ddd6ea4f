"""Which prompts are taken in chunks, by the figures at the rule, told by the workspace (no GPU needed)."""
import ctypes

import pytest

from flagdnn_b200 import _native as nat


@pytest.mark.parametrize("dtype,dk,least", [(nat.BF16, 128, 12), (nat.F16, 64, 12), (nat.F32, 64, 12), (nat.F32, 65, 17), (nat.F32, 128, 17)])
def test_short_prompts_go_token_by_token(native_lib, dtype, dk, least):
    def scratch(length, keys=dk):
        d, nbytes = nat.DeltaRuleDesc(), ctypes.c_int64()
        d.dtype = d.gate_dtype = dtype
        d.n, d.l, d.key_heads, d.heads, d.dk, d.dv = 2, length, 2, 4, keys, 64
        nat.check(native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
        return nbytes.value

    assert scratch(least - 1) == 0 and scratch(least) > 0 and scratch(least) == scratch(64)
    assert scratch(1000, 129) == 0
