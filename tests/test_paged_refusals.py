"""The argument checks of the rotary and paged entries, and the frequency
tables, without a GPU: arguments are checked before the device is looked for,
so a faulty call names its fault anywhere and a sound one names the device."""
import ctypes as C
import math

import numpy as np
import pytest

import aigpu
from oracle import oracle as O

PTR = 1 << 20      # stands for device memory: no check reads through it


def _refused(entry, args, why):
    if aigpu.available():
        pytest.skip("the pointers stand for nothing: no call is made beside a device")
    assert getattr(aigpu.lib(), entry)(C.byref(args)) == 0
    assert why in aigpu.last_error(), aigpu.last_error()


def _cache(**kw):
    base = dict(keys=PTR, values=PTR, table=PTR, lengths=PTR, batch=3, pages=10, pageSize=16, kvHeads=2, dim=128,
                tableWidth=5)
    return aigpu.AiGpuPagedCache(**{**base, **kw})


def _rotary(**kw):
    base = dict(x=PTR, out=4 * PTR, positions=PTR, frequencies=PTR, rotaryDims=64, count=4, heads=2, dim=64)
    return aigpu.AiGpuRotary(**{**base, **kw})


def _append(cache=None, **kw):
    base = dict(cache=cache or _cache(), k=PTR, v=PTR, rotaryFrequencies=PTR, rotaryDims=128, count=3)
    return aigpu.AiGpuPagedAppend(**{**base, **kw})


def _decode(cache=None, **kw):
    base = dict(cache=cache or _cache(), q=PTR, out=2 * PTR, rotaryFrequencies=PTR, rotaryDims=128, maxLength=80, heads=4)
    return aigpu.AiGpuPagedDecode(**{**base, **kw})


@pytest.mark.parametrize("change,why", [
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(frequencies=None), "null"),
    (dict(type=2), "type"), (dict(dim=0), "dim"), (dict(heads=65536), "heads"),
    (dict(rotaryDims=0), "rotaryDims"), (dict(rotaryDims=63), "rotaryDims"), (dict(rotaryDims=66), "rotaryDims"),
    (dict(amplitude=-1.0), "amplitude"), (dict(amplitude=math.inf), "amplitude"),
    (dict(amplitude=math.nan), "amplitude"), (dict(positions=None, start=2 ** 32 - 3), "positions"),
    (dict(positions=None, start=2 ** 64 - 2), "positions"), (dict(count=2 ** 40), "positions"),
    (dict(tokenStride=2 ** 41), "stride"), (dict(outHeadStride=32), "overlap"), (dict(outTokenStride=100), "overlap"),
    (dict(out=PTR + 16), "overlaps"), (dict(out=PTR, outTokenStride=256), "overlaps"),
    (dict(x=PTR + 2), "aligned"), (dict(type=1, out=4 * PTR + 1), "aligned"),
])
def test_rotary_refuses(change, why):
    _refused("aigpu_rotary", _rotary(**change), why)


@pytest.mark.parametrize("change,why", [
    (dict(keys=None), "null"), (dict(values=None), "null"), (dict(table=None), "null"), (dict(lengths=None), "null"),
    (dict(dim=80), "dim"), (dict(dim=512), "dim"), (dict(dim=0), "pool"), (dict(kvHeads=0), "pool"),
    (dict(pages=0), "pool"), (dict(pages=2 ** 31), "range"), (dict(batch=2 ** 20 + 1), "range"),
    (dict(pageSize=0), "pageSize"), (dict(pageSize=2 ** 25), "pageSize"), (dict(tableWidth=0), "tableWidth"),
    (dict(tableStride=2 ** 50), "tableStride"), (dict(keys=PTR + 8), "aligned"),
    (dict(pageStride=4096, headStride=2048, rowStride=132), "multiples"),
    (dict(pageStride=4096, headStride=2048, rowStride=64), "overlap"),
    (dict(pageStride=2 ** 62, headStride=2048, rowStride=128), "range"),
])
def test_the_cache_is_checked_by_both_entries(change, why):
    _refused("aigpu_paged_append", _append(_cache(**change)), why)
    _refused("aigpu_paged_decode", _decode(_cache(**change)), why)
    assert aigpu.lib().aigpu_paged_decode_workspace(C.byref(_decode(_cache(**change)))) == 0


@pytest.mark.parametrize("change,why", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(inType=2), "type"), (dict(count=4), "one token"),
    (dict(count=2 ** 31, starts=PTR), "many"), (dict(kStride=255), "overlap"), (dict(vStride=8), "overlap"),
    (dict(kStride=2 ** 41), "range"), (dict(rotaryDims=0), "rotaryDims"), (dict(rotaryDims=129), "rotaryDims"),
    (dict(rotaryDims=2 ** 31 + 2), "rotaryDims"), (dict(amplitude=-0.5), "amplitude"), (dict(k=PTR + 2), "aligned"),
])
def test_append_refuses(change, why):
    _refused("aigpu_paged_append", _append(**change), why)


def test_append_needs_rows_of_their_own():
    """pages that share rows are read by a decode, but two tokens would be written to one place"""
    for shared in (dict(pageStride=0, headStride=2048, rowStride=128), dict(pageStride=2048, headStride=0, rowStride=128),
                   dict(pageStride=4096, headStride=1024, rowStride=128),
                   dict(pageStride=2048, headStride=2048, rowStride=128)):
        _refused("aigpu_paged_append", _append(_cache(**shared)), "overlap")
        _refused("aigpu_paged_decode", _decode(_cache(**shared)), "no usable gfx950 device")
    for apart in (dict(pageStride=4096, headStride=128, rowStride=256), dict(pageStride=8192, headStride=4096, rowStride=256),
                  dict(pageStride=128, headStride=1280, rowStride=2560), dict(pageStride=16, headStride=0, rowStride=128, pages=1, kvHeads=1)):
        _refused("aigpu_paged_append", _append(_cache(**apart)), "no usable gfx950 device")


@pytest.mark.parametrize("change,why", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(inType=7), "type"), (dict(heads=0), "heads"),
    (dict(heads=5), "heads"), (dict(heads=2 ** 17), "heads"), (dict(qStride=64), "qStride"),
    (dict(outputGate=1), "gate"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(maxLength=81), "maxLength"), (dict(rotaryDims=130), "rotaryDims"), (dict(amplitude=math.inf), "amplitude"),
    (dict(qTokenStride=2 ** 41), "range"), (dict(q=PTR + 2), "aligned"), (dict(out=PTR), "overlaps"),
    (dict(out=PTR + 4 * 128 * 11), "overlaps"), (dict(maxLength=2 ** 31 + 1), "maxLength"),
    (dict(workspace=PTR + 64, workspaceBytes=1 << 40), "aligned"),
])
def test_decode_refuses(change, why):
    _refused("aigpu_paged_decode", _decode(**change), why)


@pytest.mark.parametrize("entry", ["aigpu_rotary", "aigpu_paged_append", "aigpu_paged_decode",
                                   "aigpu_paged_decode_workspace"])
def test_null_arguments(entry):
    assert getattr(aigpu.lib(), entry)(None) == 0
    assert "null" in aigpu.last_error()


def test_sound_calls_miss_only_the_device():
    for entry, args in (("aigpu_rotary", _rotary()), ("aigpu_paged_append", _append()),
                        ("aigpu_paged_decode", _decode()),
                        ("aigpu_rotary", _rotary(out=PTR)),                                     # in place
                        ("aigpu_rotary", _rotary(tokenStride=512, outTokenStride=512, out=PTR + 512)),   # side by side
                        ("aigpu_rotary", _rotary(headStride=256, outHeadStride=256, tokenStride=64,
                                                 outTokenStride=64))):                         # head-major
        _refused(entry, args, "no usable gfx950 device")


def test_wrappers_refuse_host_tensors():
    import torch
    x = torch.zeros((2, 2, 64))
    pages = torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        aigpu.rotary(x, x, torch.zeros(32))
    with pytest.raises(ValueError):
        aigpu.paged_append(x, x, pages, pages, i[None], i)
    with pytest.raises(ValueError):
        aigpu.paged_decode(x, x, pages, pages, i[None], i)
    with pytest.raises(TypeError):
        aigpu.rotary(np.zeros((2, 2, 64)), x, x)


def _here(t):
    """t, saying that it lies on the backend's device"""
    import torch

    class Here(torch.Tensor):
        def get_device(self):
            return 0
    return t.as_subclass(Here)


def test_wrappers_refuse_broadcast_tables_and_pages():
    """a row stride of 0 means the dense one to the entries, which lies past what a broadcast view holds"""
    import torch
    if aigpu.available():
        pytest.skip("the tensors are the host's: no call is made beside a device")
    aigpu._with_torch()
    pages = _here(torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16))
    row = _here(torch.zeros((4, 2, 16, 1), dtype=torch.bfloat16)[:1, :1, :1].expand(1, 1, 1, 64))
    one = _here(torch.zeros(64, dtype=torch.bfloat16).expand(4, 2, 16, 64))
    table, lengths = _here(torch.zeros((3, 5), dtype=torch.int32)), _here(torch.zeros(3, dtype=torch.int32))
    shared = _here(torch.zeros((1, 5), dtype=torch.int32).expand(3, 5))
    with pytest.raises(ValueError, match="broadcast"):
        aigpu._paged_cache(pages, pages, shared, lengths)
    with pytest.raises(ValueError, match="broadcast"):
        aigpu._paged_cache(one, one, table, lengths)
    with pytest.raises(ValueError, match="unit stride"):
        aigpu._paged_cache(row, row, table, lengths)
    assert aigpu._paged_cache(pages, pages, table, lengths)[-4:] == (5, 2048, 1024, 64)


def test_a_workspace_for_a_refused_call_is_refused():
    import torch
    if aigpu.available():
        pytest.skip("the tensors are the host's: no call is made beside a device")
    pages = _here(torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16))
    table, lengths = _here(torch.zeros((3, 5), dtype=torch.int32)), _here(torch.zeros(3, dtype=torch.int32))
    q, out = _here(torch.zeros((3, 4, 64))), _here(torch.zeros((3, 4, 64)))
    aigpu._with_torch()
    with pytest.raises(aigpu.AiGpuError, match="maxLength"):
        aigpu.paged_decode_workspace(q, out, pages, pages, table, lengths, max_length=81)


# ----------------------------------------------------------------- frequency tables
def test_frequencies_of_the_shared_kinds():
    """the oracle forms them in fp32: a power (2 ulp), a division, and for llama3 the wave's (4 roundings through a
    blend whose slope is at most low..high's width) - 16 half steps cover it"""
    for dims in (2, 64, 96, 128):
        for kind, name in ((0, "none"), (1, "linear"), (2, "llama3")):
            want = O.rotary_frequencies(dims, 5e5, kind, factor=8.0, low=1.0, high=4.0, original=8192.0)
            got, amplitude = aigpu.rotary_frequencies(dims, 5e5, name, factor=8.0, original=8192.0, low=1.0, high=4.0)
            assert amplitude == 1.0
            assert (np.abs(got - want) <= 16 * 2.0 ** -24 * want).all()


def test_frequencies_ntk():
    """the base grows so that the slowest pair turns `factor` times slower and the fastest as before"""
    got, _ = aigpu.rotary_frequencies(128, 1e4, "ntk", factor=4.0)
    plain, _ = aigpu.rotary_frequencies(128, 1e4)
    assert got[0] == plain[0] == 1.0
    assert abs(got[-1] * 4 / plain[-1] - 1) <= 4 * 2.0 ** -24
    assert (np.diff(got / plain) < 0).all()


def test_frequencies_yarn():
    """fast pairs kept, slow pairs divided, a straight ramp between the two pair indices"""
    dims, base, factor, original = 128, 1e6, 8.0, 4096.0
    got, amplitude = aigpu.rotary_frequencies(dims, base, "yarn", factor=factor, original=original)
    assert amplitude == np.float32(0.1 * math.log(factor) + 1.0)
    f = base ** (-np.arange(dims // 2) * 2.0 / dims)
    turns = original * f / (2 * math.pi)
    assert np.array_equal(got[turns > 34], f.astype(np.float32)[turns > 34])
    slow = turns < 0.75
    assert slow.any() and (np.abs(got[slow] - f[slow] / factor) <= 2.0 ** -24 * f[slow]).all()
    share = (f - got) / (f - f / factor)
    inside = share[(share > 0.01) & (share < 0.99)]
    assert len(inside) > 4 and np.abs(np.diff(inside, 2)).max() < 1e-5
    one, a = aigpu.rotary_frequencies(dims, base, "yarn", factor=1.0, original=original)
    assert a == 1.0 and np.abs(one / f - 1).max() <= 2 * 2.0 ** -24


@pytest.mark.parametrize("args", [
    dict(rotary_dims=63, theta=1e4), dict(rotary_dims=0, theta=1e4), dict(rotary_dims=64, theta=1.0),
    dict(rotary_dims=64, theta=math.inf), dict(rotary_dims=64, theta=1e4, scaling="linear", factor=0.5),
    dict(rotary_dims=64, theta=1e4, scaling="linear", factor=math.nan),
    dict(rotary_dims=2, theta=1e4, scaling="ntk", factor=2.0),
    dict(rotary_dims=64, theta=1e4, scaling="llama3", factor=2.0, original=0.0),
    dict(rotary_dims=64, theta=1e4, scaling="llama3", factor=2.0, original=8192.0, low=4.0, high=4.0),
    dict(rotary_dims=64, theta=1e4, scaling="yarn", factor=2.0, original=math.nan),
])
def test_frequencies_refused(args):
    with pytest.raises(aigpu.AiGpuError):
        aigpu.rotary_frequencies(**args)


def test_struct_layouts(tmp_path):
    """the ctypes structures and the packed forms have the header's layout"""
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                          "aigpu_attention.h")
    structs = {c.__name__: c for c in (aigpu.AiGpuRotary, aigpu.AiGpuRotaryScaling, aigpu.AiGpuPagedCache,
                                       aigpu.AiGpuPagedAppend, aigpu.AiGpuPagedDecode)}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        cls = structs[name]
        assert (C.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), (name, field)
    for name, cls in (("aigpu_rotary", aigpu.AiGpuRotary), ("aigpu_paged_append", aigpu.AiGpuPagedAppend),
                      ("aigpu_paged_decode", aigpu.AiGpuPagedDecode)):
        packed = aigpu._PACK[name]
        assert packed.size == C.sizeof(cls)
        # each value lands in the field of its place
        flat = [f for f, t in cls._fields_ if f != "cache"]
        if cls is not aigpu.AiGpuRotary:
            flat = [f for f, _ in aigpu.AiGpuPagedCache._fields_] + flat
        a = cls.from_buffer_copy(packed.pack(*range(1, len(flat) + 1)))
        for i, f in enumerate(flat):
            assert getattr(a if hasattr(a, f) else a.cache, f) == i + 1, f


def test_values_out_of_range_are_refused_not_wrapped():
    for bad in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            aigpu._packed("aigpu_paged_decode", *([0] * 24 + [bad] + [0] * 10))
