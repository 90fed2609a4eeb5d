"""Overlapping arrays of the verification dispatches are refused; tried without a GPU, since descriptors are checked before
the context is looked at."""
import pytest

from .test_verify_ops_cpu import f16_cache, int8_cache, refusal

FAR = 1 << 45


@pytest.mark.parametrize("apart,fine", [(2, False), (254, False), (256, True)])
def test_rows_that_end_past_64_bits(capi, apart, fine):
    desc = capi.KvReadDesc(tokens=(1 << 31) - 1, out_stride=(1 << 32) - 1, k_out=FAR, v_out=FAR + apart, slots=0x5000, cache=int8_cache(capi))
    why = refusal(capi, "ztvm_kv_read", desc)[1]
    assert why == "null context" if fine else "overlap" in why, why
