"""The argument checks of packed attention, scored decodes and the 4-bit cache, and
the layouts of their structures, without a GPU: arguments are checked before the
device is looked for, so a faulty call names its fault anywhere and a sound one
names the device."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import aigpu
from paged_q4_util import BLOCK, MOST, encode64, values64
from test_paged_refusals import PTR, _decode, _here

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "aigpu_attention.h")


def _refused(entry, why, *args):
    if aigpu.available():
        pytest.skip("the pointers stand for nothing: no call is made beside a device")
    assert getattr(aigpu.lib(), entry)(*(C.byref(a) if a is not None else None for a in args)) == 0
    assert why in aigpu.last_error(), aigpu.last_error()


def _cache(**kw):
    base = dict(keyCodes=PTR, valueCodes=PTR, keyScales=PTR, valueScales=PTR, table=PTR, lengths=PTR, batch=3, pages=10,
                pageSize=16, kvHeads=2, dim=128, tableWidth=5)
    return aigpu.AiGpuPagedCacheQ4(**{**base, **kw})


def _append(cache=None, **kw):
    base = dict(cache=cache or _cache(), k=PTR, v=PTR, rotaryFrequencies=PTR, rotaryDims=128, count=3)
    return aigpu.AiGpuPagedAppendQ4(**{**base, **kw})


def _read(cache=None, **kw):
    base = dict(cache=cache or _cache(), k=PTR, v=2 * PTR, count=3)
    return aigpu.AiGpuPagedReadQ4(**{**base, **kw})


def _decode4(cache=None, **kw):
    base = dict(cache=cache or _cache(), q=PTR, out=2 * PTR, rotaryFrequencies=PTR, rotaryDims=128, maxLength=80, heads=4)
    return aigpu.AiGpuPagedDecodeQ4(**{**base, **kw})


def _packed(**kw):
    base = dict(q=PTR, k=2 * PTR, v=3 * PTR, out=4 * PTR, starts=PTR, inType=1, outType=1, count=50, keyCount=50,
                documents=3, heads=4, kvHeads=2, dim=128)
    return aigpu.AiGpuPackedAttention(**{**base, **kw})


@pytest.mark.parametrize("change,why", [
    (dict(keyCodes=None), "null"), (dict(valueCodes=None), "null"), (dict(keyScales=None), "null"),
    (dict(valueScales=None), "null"), (dict(table=None), "null"), (dict(lengths=None), "null"),
    (dict(dim=80), "dim"), (dict(dim=512), "dim"), (dict(dim=0), "pool"), (dict(kvHeads=0), "pool"),
    (dict(pages=0), "pool"), (dict(pages=2 ** 31), "range"), (dict(batch=2 ** 20 + 1), "range"),
    (dict(pageSize=0), "pageSize"), (dict(pageSize=2 ** 25), "pageSize"), (dict(tableWidth=0), "tableWidth"),
    (dict(tableStride=2 ** 50), "tableStride"), (dict(keyCodes=PTR + 8), "aligned"),
    (dict(valueScales=PTR + 4), "aligned"), (dict(pageStride=64, headStride=16, rowStride=0), "overlap"),
    (dict(pageStride=2 ** 62, headStride=16, rowStride=1), "range"),
])
def test_the_cache_is_checked_by_all_entries(change, why):
    _refused("aigpu_paged_append_q4", why, _append(_cache(**change)))
    _refused("aigpu_paged_read_q4", why, _read(_cache(**change)))
    _refused("aigpu_paged_decode_q4", why, _decode4(_cache(**change)))
    assert aigpu.lib().aigpu_paged_decode_q4_workspace(C.byref(_decode4(_cache(**change)))) == 0


@pytest.mark.parametrize("change,why", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(inType=2), "type"), (dict(count=4), "one token"),
    (dict(count=2 ** 31, starts=PTR), "many"), (dict(kStride=255), "overlap"), (dict(vStride=8), "overlap"),
    (dict(kStride=2 ** 41), "range"), (dict(rotaryDims=0), "rotaryDims"), (dict(rotaryDims=129), "rotaryDims"),
    (dict(rotaryDims=2 ** 31 + 2), "rotaryDims"), (dict(amplitude=-0.5), "amplitude"), (dict(k=PTR + 2), "aligned"),
])
def test_append_refuses(change, why):
    _refused("aigpu_paged_append_q4", why, _append(**change))


def test_append_needs_rows_of_their_own():
    for shared in (dict(pageStride=0, headStride=16, rowStride=1), dict(pageStride=32, headStride=0, rowStride=1),
                   dict(pageStride=32, headStride=8, rowStride=1), dict(pageStride=16, headStride=16, rowStride=1)):
        _refused("aigpu_paged_append_q4", "overlap", _append(_cache(**shared)))
        _refused("aigpu_paged_decode_q4", "no usable gfx950 device", _decode4(_cache(**shared)))
    for apart in (dict(pageStride=32, headStride=1, rowStride=2), dict(pageStride=64, headStride=32, rowStride=2),
                  dict(pageStride=1, headStride=10, rowStride=20)):
        _refused("aigpu_paged_append_q4", "no usable gfx950 device", _append(_cache(**apart)))


@pytest.mark.parametrize("change,why", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(outType=2), "type"), (dict(count=4), "one token"),
    (dict(count=2 ** 31, starts=PTR), "many"), (dict(kStride=255), "overlap"), (dict(vStride=2 ** 41), "range"),
    (dict(k=PTR + 2), "aligned"), (dict(v=PTR), "overlap"), (dict(v=PTR + 4 * 128), "overlap"),
])
def test_read_refuses(change, why):
    _refused("aigpu_paged_read_q4", why, _read(**change))


def test_read_takes_slices_of_the_same_rows():
    _refused("aigpu_paged_read_q4", "no usable gfx950 device", _read(kStride=512, vStride=512, v=PTR + 4 * 256))


@pytest.mark.parametrize("change,why", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(inType=7), "type"), (dict(heads=0), "heads"),
    (dict(heads=5), "heads"), (dict(heads=2 ** 17), "heads"), (dict(qStride=64), "qStride"),
    (dict(outputGate=1), "gate"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(maxLength=81), "maxLength"), (dict(rotaryDims=130), "rotaryDims"), (dict(amplitude=math.inf), "amplitude"),
    (dict(qTokenStride=2 ** 41), "range"), (dict(q=PTR + 2), "aligned"), (dict(out=PTR), "overlaps"),
    (dict(maxLength=2 ** 31 + 1), "maxLength"), (dict(workspace=PTR + 64, workspaceBytes=1 << 40), "aligned"),
    (dict(workspace=PTR, workspaceBytes=16), "holds"), (dict(cap=-1.0), "cap"), (dict(cap=math.inf), "cap"),
    (dict(cap=math.nan), "cap"), (dict(cap=1e-8), "cap"), (dict(slopes=PTR + 2), "slopes"),
])
def test_decode_refuses(change, why):
    _refused("aigpu_paged_decode_q4", why, _decode4(**change))


@pytest.mark.parametrize("change,why", [
    (dict(cap=-1.0), "cap"), (dict(cap=math.nan), "cap"), (dict(cap=1e7), "cap"), (dict(slopes=PTR + 1), "slopes"),
])
def test_scored_decode_refuses(change, why):
    _refused("aigpu_paged_decode_scored", why, _decode(), aigpu.AiGpuScores(**change))


def test_scored_decode_checks_its_call_too():
    _refused("aigpu_paged_decode_scored", "null", _decode(), None)
    _refused("aigpu_paged_decode_scored", "null", None, aigpu.AiGpuScores(cap=1.0))
    _refused("aigpu_paged_decode_scored", "heads", _decode(heads=5), aigpu.AiGpuScores(cap=1.0))
    _refused("aigpu_paged_decode_scored", "no usable gfx950 device", _decode(), aigpu.AiGpuScores())
    _refused("aigpu_paged_decode_scored", "no usable gfx950 device", _decode(), aigpu.AiGpuScores(cap=30.0, slopes=PTR))


@pytest.mark.parametrize("change,why", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"),
    (dict(inType=2), "type"), (dict(outType=3), "type"), (dict(dim=80), "dim"), (dict(heads=0), "heads"),
    (dict(heads=5), "heads"), (dict(kvHeads=0), "heads"), (dict(heads=2 ** 17), "range"), (dict(count=2 ** 31), "range"),
    (dict(keyCount=2 ** 31, keyStarts=PTR), "range"), (dict(documents=2 ** 25), "range"),
    (dict(starts=None), "one document"), (dict(starts=None, documents=1, keyStarts=PTR), "keyStarts"),
    (dict(keyCount=60), "as many keys"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(cap=-2.0), "cap"), (dict(cap=math.nan), "cap"), (dict(cap=1e-7), "cap"), (dict(q=PTR + 8), "aligned"),
    (dict(k=PTR + 2), "aligned"), (dict(vTokenStride=260), "aligned"), (dict(qHeadStride=129), "aligned"),
    (dict(out=4 * PTR + 1), "aligned"), (dict(prefix=PTR + 2), "aligned"), (dict(kTokenStride=2 ** 41), "range"),
    (dict(outHeadStride=64), "overlap"), (dict(outTokenStride=100), "overlap"), (dict(out=PTR), "overlaps"),
    (dict(out=2 * PTR + 4096), "overlaps"), (dict(out=3 * PTR - 4096), "overlaps"),
    (dict(count=2 ** 28, keyCount=2 ** 28, heads=64, kvHeads=2, q=1 << 50, k=1 << 52, v=1 << 54, out=1 << 56), "many"),
    (dict(workspace=PTR + 64, workspaceBytes=1 << 40), "aligned"),
    (dict(count=3, keyCount=10000, keyStarts=PTR, workspace=PTR, workspaceBytes=16, k=1 << 40, v=1 << 41), "holds"),
])
def test_packed_attention_refuses(change, why):
    _refused("aigpu_packed_attention", why, _packed(**change))


def test_a_scale_that_leaves_no_number_over_the_cap():
    for scale, cap in ((1e33, 1e-6), (1e-38, 1e6)):
        _refused("aigpu_packed_attention", "suit", _packed(scale=scale, cap=cap))
        _refused("aigpu_paged_decode_scored", "suit", _decode(scale=scale), aigpu.AiGpuScores(cap=cap))


def test_more_workgroups_than_a_launch_has():
    _refused("aigpu_packed_attention", "many", _packed(documents=2 ** 24))
    _refused("aigpu_packed_attention", "no usable gfx950 device", _packed(documents=2 ** 20))


def test_sound_calls_miss_only_the_device():
    lattice = dict(qTokenStride=12 * 128, kTokenStride=12 * 128, vTokenStride=12 * 128, outTokenStride=12 * 128)
    row = 2 * 128
    for args in (_packed(), _packed(starts=None, documents=1), _packed(keyCount=90, keyStarts=PTR),
                 _packed(cap=50.0, slopes=PTR, prefix=PTR, window=7), _packed(inType=0, outType=0),
                 _packed(count=0, keyCount=0), _packed(documents=0),
                 # q, k, v and out as slices of the same rows
                 _packed(q=PTR, k=PTR + 4 * row, v=PTR + 6 * row, out=PTR + 8 * row, **lattice)):
        _refused("aigpu_packed_attention", "no usable gfx950 device", args)
    for entry, args in (("aigpu_paged_append_q4", _append()), ("aigpu_paged_read_q4", _read()),
                        ("aigpu_paged_decode_q4", _decode4(cap=30.0, slopes=PTR, window=9))):
        _refused(entry, "no usable gfx950 device", args)


@pytest.mark.parametrize("entry", ["aigpu_paged_append_q4", "aigpu_paged_read_q4", "aigpu_paged_decode_q4",
                                   "aigpu_paged_decode_q4_workspace", "aigpu_packed_attention"])
def test_null_arguments(entry):
    assert getattr(aigpu.lib(), entry)(None) == 0
    assert "null" in aigpu.last_error()


def test_workspaces():
    """few tokens over many keys have their keys split; a refused call has no size"""
    size = aigpu.lib().aigpu_packed_attention_workspace
    size.restype = C.c_uint64
    assert size(None) == 2 ** 64 - 1
    assert size(C.byref(_packed(dim=80))) == 2 ** 64 - 1
    assert size(C.byref(_packed(count=2 ** 20, keyCount=2 ** 20, k=1 << 40, v=1 << 42, out=1 << 44))) == 0
    few = size(C.byref(_packed(count=3, keyCount=10000, keyStarts=PTR, k=1 << 40, v=1 << 41)))
    assert few > 0 and few % ((128 + 2) * 128 * 4) == 0
    assert aigpu.lib().aigpu_paged_decode_q4_workspace(C.byref(_decode4())) > 0


STRUCTS = {n: getattr(aigpu, n) for n in ("AiGpuScores", "AiGpuPagedCacheQ4", "AiGpuPagedAppendQ4", "AiGpuPagedReadQ4",
                                          "AiGpuPagedDecodeQ4", "AiGpuPackedAttention")}


def test_struct_layouts_match_the_c_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        cls = STRUCTS[name]
        assert (C.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), line
    # the wrappers pack the structures themselves
    for entry, cls in (("aigpu_paged_append_q4", "AiGpuPagedAppendQ4"), ("aigpu_paged_read_q4", "AiGpuPagedReadQ4"),
                       ("aigpu_paged_decode_q4", "AiGpuPagedDecodeQ4"), ("scores", "AiGpuScores"),
                       ("aigpu_packed_attention", "AiGpuPackedAttention")):
        assert aigpu._PACK[entry].size == C.sizeof(STRUCTS[cls]), entry


def _pools(dim=64, pages=4, kv=2, size=16):
    import torch
    codes = [_here(torch.zeros((pages, kv, size, dim // 2), dtype=torch.uint8)) for _ in "kv"]
    scales = [_here(torch.zeros((pages, kv, size, dim // 32), dtype=torch.float16)) for _ in "kv"]
    return [codes[0], scales[0], codes[1], scales[1], _here(torch.zeros((3, 5), dtype=torch.int32)),
            _here(torch.zeros(3, dtype=torch.int32))]


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    import torch
    if aigpu.available():
        pytest.skip("the tensors are the host's: no call is made beside a device")
    x, out = _here(torch.zeros((3, 4, 64))), _here(torch.zeros((3, 4, 64)))
    k = _here(torch.zeros((3, 2, 64)))
    pools = _pools()
    host = [p.as_subclass(torch.Tensor) for p in pools]
    with pytest.raises(ValueError, match="cuda:0"):
        aigpu.paged_append_q4(k, k, *host)
    with pytest.raises(ValueError, match="cuda:0"):
        aigpu.packed_attention(x.as_subclass(torch.Tensor), k, k, out)
    for at, wrong, error in ((0, torch.int8, TypeError), (1, torch.bfloat16, TypeError), (4, torch.int64, TypeError),
                             (5, torch.int64, TypeError)):
        bad = list(pools)
        bad[at] = _here(bad[at].as_subclass(torch.Tensor).to(wrong))
        with pytest.raises(error):
            aigpu.paged_read_q4(k, k.clone(), *bad)
    bad = list(pools)
    bad[1] = _here(torch.zeros((4, 2, 16, 4), dtype=torch.float16))
    with pytest.raises(ValueError, match="dim / 32"):
        aigpu.paged_decode_q4(x, out, *bad)
    bad = list(pools)
    bad[2] = _here(torch.zeros((4, 16, 2, 32), dtype=torch.uint8).transpose(1, 2))
    with pytest.raises(ValueError, match="same strides"):
        aigpu.paged_decode_q4(x, out, *bad)
    bad = list(pools)
    bad[0] = _here(torch.zeros((4, 2, 16, 40), dtype=torch.uint8)[..., :32])
    with pytest.raises(ValueError, match="dense"):
        aigpu.paged_decode_q4(x, out, *bad)
    with pytest.raises(ValueError, match="elements"):
        aigpu.paged_decode_q4(x, out, *pools, slopes=_here(torch.zeros(3)), stream=0)
    with pytest.raises(ValueError, match="entries"):
        aigpu.packed_attention(x, k, k, out, starts=_here(torch.zeros(3, dtype=torch.int32)),
                               key_starts=_here(torch.zeros(4, dtype=torch.int32)))
    with pytest.raises(ValueError, match="broadcast"):
        aigpu.packed_attention(x, _here(torch.zeros((1, 2, 64)).expand(3, 2, 64)), k, out)
    with pytest.raises(aigpu.AiGpuError, match="no usable gfx950 device"):
        aigpu.packed_attention(x, k, k.clone(), out.clone(), stream=0)
    with pytest.raises(aigpu.AiGpuError, match="overlaps"):
        aigpu.packed_attention(x, k, k, x, stream=0)
    with pytest.raises(aigpu.AiGpuError, match="no usable gfx950 device"):
        aigpu.paged_decode_q4(x, out, *pools, stream=0)


def test_wrappers_take_strided_pools():
    """key and value rows of one buffer, heads of a position together, dimensions of one of any stride"""
    import torch
    if aigpu.available():
        pytest.skip("the tensors are the host's: no call is made beside a device")
    both = torch.zeros((4, 2, 3, 16, 32), dtype=torch.uint8), torch.zeros((4, 2, 3, 16, 2), dtype=torch.float16)
    pools = [_here(t[:, i]) for i in (0, 1) for t in both] + _pools()[4:]
    assert aigpu._paged_cache_q4(*pools)[-3:] == (96, 16, 1)
    turned = [_here(t.as_subclass(torch.Tensor).transpose(1, 2).contiguous().transpose(1, 2)) for t in _pools(kv=3)[:4]]
    assert aigpu._paged_cache_q4(*turned, *_pools()[4:])[-3:] == (48, 1, 3)
    one = [_here(t.as_subclass(torch.Tensor)[:1, :1, :1].as_strided((1, 1, 1, t.shape[3]), (7, 5, 3, 1))) for t in _pools()[:4]]
    assert aigpu._paged_cache_q4(*one, *_pools()[4:])[-3:] == (1, 1, 1)
    with pytest.raises(ValueError, match="broadcast"):
        aigpu._paged_cache_q4(*[_here(t.as_subclass(torch.Tensor)[:, :, :1].expand(4, 2, 16, t.shape[3]))
                                for t in _pools()[:4]], *_pools()[4:])


def test_the_codes_of_rows():
    """the tests' own encoding: the nearest of the fifteen values, a scale that no smaller one of 8 bits replaces"""
    r = np.random.default_rng(1)
    for size in (1e-7, 1e-3, 1.0, 300.0, 1e5):
        x = size * r.standard_normal((50, 64))
        codes, scales = encode64(x)
        held = values64(codes, scales)
        wide = np.repeat(scales, BLOCK, -1)
        assert (codes >= 1).all() and (codes <= 15).all()
        inside = np.abs(x) <= 7 * MOST
        assert (np.abs(x - held)[inside] <= wide[inside] / 2 * (1 + 1e-12)).all()
        assert (scales.astype(np.float16) == scales).all() and (scales <= MOST).all()
        top = np.abs(x).reshape(50, 2, BLOCK).max(-1)
        m, e = np.frexp(scales)
        bits = m * 256
        assert (bits == np.rint(bits)).all()
        below = scales - np.ldexp(1.0, np.maximum(e - 8, -24))
        free = scales < MOST
        assert (7 * scales >= top)[free].all() and (7 * below < top)[free].all()
    codes, scales = encode64(np.array([[0.5, -0.5, 1.5, 7.0] + [0.0] * 28]))
    assert scales[0, 0] == 1.0 and codes[0, :4].tolist() == [9, 8, 10, 15]
    codes, scales = encode64(np.array([[np.nan] + [1.0] * 31, [0.0] * 32]))
    assert np.isnan(scales[0, 0]) and scales[1, 0] == 0 and (codes == 8).all()
