"""The no-device backend refuses a packed attention's workspace query as it refuses the call."""
import ctypes as C

import aigpu


def test_the_stub_refuses_the_query_as_the_call():
    stub = aigpu.load_library(aigpu.STUB)
    args = aigpu.AiGpuPackedAttention(inType=1, outType=1, count=50, keyCount=50, documents=1, heads=4, kvHeads=2, dim=128)
    assert stub.aigpu_packed_attention(C.byref(args)) == 0
    # 0 would say that the call needs no workspace
    assert stub.aigpu_packed_attention_workspace(C.byref(args)) == 2 ** 64 - 1
    assert b"no device" in stub.aigpu_last_error()
