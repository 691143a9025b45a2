"""The argument checks of spmm24_launch_moe and its workspace size, on the CPU
(no GPU work is reached)."""
import ctypes

import pytest

import spmm24

OK = dict(tokens=3, hidden=256, inter=128, experts=8, top_k=2, activation=2, norm_topk=1, x=0x10000, router=0x20000,
          gate_up=0x30000, gate_up_meta=0x40000, down=0x50000, down_meta=0x60000, topk_ids=0x70000,
          topk_weights=0x80000, y=0x90000, workspace=0x100000, workspace_bytes=1 << 30)
INT8 = dict(flags=spmm24.MOE_INT8, gate_up_scale=0xA0000, down_scale=0xB0000)


def _launch(**kw):
    flags = kw.pop("flags", 0)
    layer = spmm24.MoeLayer(**(OK | kw))
    return spmm24._lib.spmm24_launch_moe(None, ctypes.byref(layer), flags)


@pytest.mark.parametrize("kw,why", [
    (dict(tokens=0), "tokens"), (dict(tokens=33), "tokens"), (dict(experts=0), "experts"), (dict(experts=257), "experts"),
    (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"), (dict(experts=32, top_k=17), "top_k"),
    (dict(hidden=96), "multiples of 64"), (dict(inter=0), "multiples of 64"), (dict(inter=-64), "multiples of 64"),
    (dict(hidden=64, **INT8), "multiples of 128"), (dict(inter=192, **INT8), "multiples of 128"),
    (dict(hidden=131072 + 64), "131072"), (dict(inter=131072 + 64), "131072"),
    (dict(tokens=32, experts=256, top_k=16, inter=16448), "32768"),
    (dict(x=0), "null"), (dict(gate_up=0), "null"), (dict(gate_up_meta=0), "null"), (dict(down=0), "null"),
    (dict(down_meta=0), "null"), (dict(y=0), "null"), (dict(workspace=0), "null"),
    (dict(x=0x10008), "16-byte"), (dict(router=0x20002), "16-byte"), (dict(gate_up=0x30004), "16-byte"),
    (dict(gate_up_meta=0x40008), "16-byte"), (dict(down=0x50001), "16-byte"), (dict(down_meta=0x60008), "16-byte"),
    (dict(topk_ids=0x70002), "4-byte"), (dict(topk_weights=0x80001), "4-byte"), (dict(y=0x90001), "2-byte"),
    (dict(router=0, topk_ids=0), "inputs"), (dict(router=0, topk_weights=0), "inputs"),
    (dict(gate_up_scale=0xA0000, down_scale=0xB0000), "scales"), (dict(gate_up_scale=0xA0000), "scales"),
    (dict(flags=spmm24.MOE_INT8), "scales"), (dict(flags=spmm24.MOE_INT8, gate_up_scale=0xA0000), "scales"),
    (dict(activation=4), "activation"), (dict(activation=-1), "activation"), (dict(flags=8), "flag"),
    (dict(flags=64), "flag"), (dict(workspace=0x100080), "256-byte"), (dict(workspace_bytes=1000), "too small"),
])
def test_refusals(kw, why):
    assert _launch(**kw) == spmm24.CUDA_ERROR_INVALID_VALUE
    assert why in spmm24._lib.spmm24_last_error().decode()


def test_epilogue_and_null_refusals():
    bad = spmm24.CUDA_ERROR_INVALID_VALUE
    assert spmm24._lib.spmm24_launch_moe(None, None, 0) == bad
    epi = spmm24.Epilogue(None, None, float("nan"), 0, 0)
    assert _launch(epilogue=ctypes.addressof(epi)) == bad
    epi = spmm24.Epilogue(None, None, 1.0, 0, spmm24.OUT_PACKED_B)
    assert _launch(epilogue=ctypes.addressof(epi), y=0x90002) == bad


def test_workspace_bytes():
    sizes = (3, 256, 128, 8, 2)
    n = spmm24.moe_workspace_bytes(*sizes)
    assert _launch(workspace_bytes=n - 1) == spmm24.CUDA_ERROR_INVALID_VALUE
    assert "too small" in spmm24._lib.spmm24_last_error().decode()
    # h of 32 tokens and 8 experts: 4 + 1 bytes for each int8 value, 2 for a 16-bit one
    big = spmm24.moe_workspace_bytes(32, 4096, 11008, 8, 2, spmm24.MOE_INT8)
    assert big - spmm24.moe_workspace_bytes(32, 4096, 11008, 8, 2) >= 32 * 8 * 11008 * 3
    for bad in ((0, 256, 128, 8, 2), (33, 256, 128, 8, 2), (3, 100, 128, 8, 2), (3, 256, 128, 8, 9)):
        with pytest.raises(ValueError):
            spmm24.moe_workspace_bytes(*bad)
    with pytest.raises(ValueError):
        spmm24.moe_workspace_bytes(3, 256, 192, 8, 2, spmm24.MOE_INT8)
