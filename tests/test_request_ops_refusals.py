"""What the per-request operators refuse, before any device work: wrong shapes and types in Python, bad sizes and
pointers at the C entries (which report an error and never raise)."""
import ctypes

import pytest
import torch

from aipu_b200 import _lib, ops

BF, F32, HF, I32, I64 = torch.bfloat16, torch.float32, torch.float16, torch.int32, torch.int64


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _adapters(**kw):
    a = dict(a=_z(2, 8, 64), b=_z(2, 32, 8), scale=_z(2, dtype=F32), ranks=_z(2, dtype=I32))
    a.update(kw)
    return ops.LoraAdapters(**a)


BAD_ADAPTERS = [
    dict(a=_z(2, 8)), dict(b=_z(32, 8)), dict(a=_z(3, 8, 64)), dict(a=_z(2, 9, 64)), dict(b=_z(2, 8, 32)),
    dict(a=_z(2, 8, 64, dtype=HF)), dict(a=_z(2, 8, 64, dtype=F32), b=_z(2, 32, 8, dtype=F32)),
    dict(scale=_z(2)), dict(scale=_z(3, dtype=F32)), dict(ranks=_z(2, dtype=I64)), dict(ranks=_z(1, dtype=I32)),
    dict(a=_z(2, 64, 8).transpose(1, 2)), dict(scale=_z(4, dtype=F32)[::2]),
]


@pytest.mark.parametrize("kw", BAD_ADAPTERS)
def test_bad_adapters(kw):
    with pytest.raises(ValueError):
        ops.lora_add(_adapters(**kw), _z(4, dtype=I32), _z(4, 64), _z(4, 32))


@pytest.mark.parametrize("ids,x,y,out", [
    (_z(4, dtype=I64), _z(4, 64), _z(4, 32), None), (_z(3, dtype=I32), _z(4, 64), _z(4, 32), None),
    (_z(8, dtype=I32)[::2], _z(4, 64), _z(4, 32), None), (_z(4, dtype=I32), _z(4, 64, dtype=F32), _z(4, 32), None),
    (_z(4, dtype=I32), _z(4, 65), _z(4, 32), None), (_z(4, dtype=I32), _z(4, 64), _z(4, 33), None),
    (_z(4, dtype=I32), _z(4, 64), _z(3, 32), None), (_z(4, dtype=I32), _z(64, 4).t(), _z(4, 32), None),
    (_z(4, dtype=I32), _z(4, 64), _z(1, 32).expand(4, 32), None), (_z(4, dtype=I32), _z(4, 64), _z(4, 32, dtype=HF), None),
    (_z(4, dtype=I32), _z(4, 64), _z(4, 32), _z(4, 32, dtype=F32)), (_z(4, dtype=I32), _z(4, 64), _z(4, 32), _z(4, 31)),
    (_z(4, dtype=I32), _z(4, 64), _z(4, 32), None)])  # the last is right but for the device
def test_bad_rows(ids, x, y, out):
    with pytest.raises(ValueError):
        ops.lora_add(_adapters(), ids, x, y, out=out)


def test_bad_projection():
    ad, ids = _adapters(a=_z(2, 8, 256)), _z(4, dtype=I32)
    w = _z(32, 144, dtype=torch.uint8)
    for args in ((0, w, 31, 256, _z(4, 256)), (0, w, 32, 512, _z(4, 256)), (0, w[:31], 32, 256, _z(4, 256)),
                 (0, w, 32, 256, _z(4, 512)[:, :256]), (0, w, 32, 256, _z(4, 256))):
        with pytest.raises(ValueError):
            ops.gemm_lora(*args, ad, ids)
    with pytest.raises(ValueError):
        ops.gemm_lora(0, w, 32, 256, _z(4, 256), ad, ids, out=_z(4, 32, dtype=F32))


GOOD = dict(tokens=_z(9, dtype=I32), spans=_z(3, 3, dtype=I64), penalties=_z(3, 3, dtype=F32), bias_begin=_z(4, dtype=I64),
            bias_ids=_z(5, dtype=I32), bias_vals=_z(5, dtype=F32), mask=_z(2, 4, dtype=I32), mask_rows=_z(3, dtype=I32))


@pytest.mark.parametrize("kw", [
    dict(tokens=None), dict(spans=None), dict(penalties=None), dict(tokens=_z(9, dtype=I64)), dict(spans=_z(3, 2, dtype=I64)),
    dict(spans=_z(3, 3, dtype=I32)), dict(spans=_z(2, 3, dtype=I64)), dict(penalties=_z(3, 3, dtype=BF)),
    dict(bias_begin=None), dict(bias_ids=None), dict(bias_vals=None), dict(bias_begin=_z(3, dtype=I64)),
    dict(bias_vals=_z(4, dtype=F32)), dict(mask=None), dict(mask_rows=None), dict(mask=_z(2, 3, dtype=I32)),
    dict(mask=_z(2, 5, dtype=I32)), dict(mask=_z(2, 4, dtype=torch.uint8)), dict(mask_rows=_z(2, dtype=I32)),
    dict(mask=_z(2, 8, dtype=I32)[:, ::2]), dict()])  # the last is right but for the device
def test_bad_controls(kw):
    with pytest.raises(ValueError):
        ops.process_logits(_z(3, 100), ops.LogitControls(**{**GOOD, **kw}))


def test_bad_logits():
    for x, out in ((_z(100), None), (_z(3, 100, dtype=HF), None), (_z(100, 3).t(), None), (_z(3, 100), _z(3, 100)),
                   (_z(3, 100), _z(3, 99, dtype=F32)), (_z(3, 100), _z(2, 100, dtype=F32))):
        with pytest.raises(ValueError):
            ops.process_logits(x, out=out)
    with pytest.raises(ValueError):
        ops.greedy_tokens(_z(3, 100))


def _lora(**kw):
    d = dict(dtype=_lib.DT_BF16, n_adapters=2, rank=8, in_features=256, out_features=32, a=16, b=16)
    d.update(kw)
    return _lib.Lora(**d)


@pytest.mark.parametrize("kw,M", [(dict(dtype=0), 4), (dict(dtype=3), 4), (dict(n_adapters=0), 4), (dict(n_adapters=32769), 4),
                                  (dict(rank=0), 4), (dict(rank=129), 4), (dict(in_features=0), 4), (dict(out_features=-1), 4),
                                  (dict(a=None), 4), (dict(b=None), 4), (dict(), -1), (dict(), 1 << 25)])
def test_c_entry_refuses_adapters(kw, M):
    L = _lib.lib()
    assert L.aipu_lora_add(None, _lora(**kw), 16, 16, 256, M, 16, 1, 32, 32, 1, 32, 16, 1 << 30, None) == _lib.AIPU_EINVAL
    assert b"bad adapters" in L.aipu_last_error()
    assert L.aipu_q4k_gemm_lora(None, 0, 16, 32, 256, 16, M, _lora(**kw), 16, 16, 256, 1 << 40, None) == _lib.AIPU_EINVAL
    assert b"bad adapters" in L.aipu_last_error()


def _add(M=300, x=16, ldx=256, y=16, ydt=1, ldy=32, out=32, odt=1, ldo=32, ws=16, n=1 << 30):
    return _lib.lib().aipu_lora_add(None, _lora(), 16, x, ldx, M, y, ydt, ldy, out, odt, ldo, ws, n, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), b"null pointer"), (dict(y=None), b"null pointer"), (dict(out=None), b"null pointer"),
    (dict(ldx=255), b"stride"), (dict(ldy=31), b"stride"), (dict(ldo=31), b"stride"), (dict(ydt=2), b"bf16, fp32"),
    (dict(ydt=1, odt=0), b"bf16, fp32"), (dict(out=16, ydt=0), b"in place"), (dict(out=16, ldo=64), b"in place"),
    (dict(ws=None), b"workspace"), (dict(ws=8), b"workspace"), (dict(n=100), b"workspace"), (dict(), b"null context")])
def test_c_entry_refuses_rows(kw, text):
    assert _add(**kw) == _lib.AIPU_EINVAL
    assert text in _lib.lib().aipu_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(wtype=4), b"bad arguments"), (dict(wtype=9), b"bad arguments"), (dict(K=128), b"bad arguments"), (dict(K=512), b"bad arguments"),
    (dict(N=31), b"bad arguments"), (dict(w=None), b"bad arguments"), (dict(x=None), b"bad arguments"), (dict(y=None), b"bad arguments"),
    (dict(w=8), b"aligned"), (dict(x=8), b"aligned"), (dict(ws=None), b"workspace"), (dict(ws=16), b"workspace"),
    (dict(n=10), b"workspace"), (dict(), b"null context")])
def test_c_entry_refuses_a_projection(kw, text):
    a = dict(wtype=0, w=16, N=32, K=256, x=16, M=4, y=16, ws=256, n=1 << 40)
    a.update(kw)
    L = _lib.lib()
    assert L.aipu_q4k_gemm_lora(None, a["wtype"], a["w"], a["N"], a["K"], a["x"], a["M"], _lora(), 16, a["y"], a["ws"], a["n"],
                                None) == _lib.AIPU_EINVAL
    assert text in L.aipu_last_error()


def test_workspace_sizes():
    L = _lib.lib()
    assert L.aipu_lora_workspace(256, 8, 64) == 0 and L.aipu_lora_workspace(16, 32768, 128) == 0
    for bad in ((-1, 8, 16), (257, 0, 16), (257, 32769, 16), (257, 8, 0), (257, 8, 129)):
        assert L.aipu_lora_workspace(*bad) == 0
    # an int per row, tiles of every adapter, and the fp32 sums of 16 ranks at least
    assert L.aipu_lora_workspace(257, 8, 3) >= 4 * 257 + 16 * 9 + 4 * 257 * 16
    assert L.aipu_q4k_gemm_lora_workspace(0, 32, 256, 3, 2, 8) >= 4 * 3 * 32
    assert L.aipu_q4k_gemm_lora_workspace(0, 32, 100, 3, 2, 8) == 0


def _process(**kw):
    a = dict(x=64, dtype=1, ld=100, M=3, V=100, ctl=None, out=128, ldo=100, token=16)
    a.update(kw)
    return _lib.lib().aipu_logits_process(None, a["x"], a["dtype"], a["ld"], a["M"], a["V"], a["ctl"], a["out"], a["ldo"],
                                          a["token"], None)


def _ctl(**kw):
    d = dict(tokens=16, n_tokens=9, spans=16, penalties=16, bias_begin=16, bias_ids=16, bias_vals=16, n_bias=5, mask=16,
             mask_rows=16, n_masks=2)
    d.update(kw)
    return _lib.LogitCtl(**d)


@pytest.mark.parametrize("kw,text", [
    (dict(M=-1), b"bad shape"), (dict(V=0), b"bad shape"), (dict(V=1 << 29, ld=1 << 29), b"bad shape"), (dict(dtype=2), b"bad shape"),
    (dict(ld=99), b"bad shape"), (dict(ldo=99), b"bad shape"), (dict(x=None), b"bad shape"), (dict(out=None, token=None), b"bad shape"),
    (dict(out=64), b"in place"), (dict(out=64, dtype=0, ld=101), b"in place"),
    (dict(ctl=_ctl(spans=None)), b"penalties need"), (dict(ctl=_ctl(penalties=None)), b"penalties need"),
    (dict(ctl=_ctl(tokens=None)), b"penalties need"), (dict(ctl=_ctl(n_tokens=-1)), b"penalties need"),
    (dict(ctl=_ctl(n_tokens=1 << 31)), b"penalties need"), (dict(ctl=_ctl(bias_ids=None)), b"biases need"),
    (dict(ctl=_ctl(bias_vals=None)), b"biases need"), (dict(ctl=_ctl(n_bias=-1)), b"biases need"),
    (dict(ctl=_ctl(mask=None)), b"masks need"), (dict(ctl=_ctl(mask_rows=None)), b"masks need"),
    (dict(ctl=_ctl(n_masks=0)), b"masks need"), (dict(ctl=_ctl()), b"null context"), (dict(), b"null context")])
def test_c_entry_refuses_logits(kw, text):
    assert _process(**kw) == _lib.AIPU_EINVAL
    assert text in _lib.lib().aipu_last_error()


@pytest.mark.parametrize("kw", [dict(a=17), dict(b=17), dict(scale=18), dict(ranks=18)])
def test_c_entries_refuse_adapters_off_their_types_alignment(kw):
    L = _lib.lib()
    assert L.aipu_lora_add(None, _lora(**kw), 16, 16, 256, 4, 16, 1, 32, 32, 1, 32, 16, 1 << 30, None) == _lib.AIPU_EINVAL
    assert b"not aligned" in L.aipu_last_error()
    assert L.aipu_q4k_gemm_lora(None, 0, 16, 32, 256, 16, 4, _lora(**kw), 16, 16, 256, 1 << 40, None) == _lib.AIPU_EINVAL
    assert b"not aligned" in L.aipu_last_error()


@pytest.mark.parametrize("kw", [dict(x=17), dict(y=17), dict(out=33), dict(y=18, ydt=0), dict(y=16, ydt=0, out=34, odt=0)])
def test_c_entry_refuses_rows_off_their_types_alignment(kw):
    assert _add(**kw) == _lib.AIPU_EINVAL
    assert b"not aligned" in _lib.lib().aipu_last_error()


@pytest.mark.parametrize("kw", [
    dict(x=65), dict(x=66, dtype=0), dict(out=130), dict(token=18), dict(ctl=_ctl(tokens=18)), dict(ctl=_ctl(spans=20)),
    dict(ctl=_ctl(penalties=18)), dict(ctl=_ctl(bias_begin=20)), dict(ctl=_ctl(bias_ids=18)), dict(ctl=_ctl(bias_vals=17)),
    dict(ctl=_ctl(mask=18)), dict(ctl=_ctl(mask_rows=18))])
def test_c_entry_refuses_logits_off_their_types_alignment(kw):
    assert _process(**kw) == _lib.AIPU_EINVAL
    assert b"not aligned" in _lib.lib().aipu_last_error()


def test_structs_match_the_header():
    """Field for field in the header's order (all 8-byte fields but the adapters' first two)."""
    assert ctypes.sizeof(_lib.Lora) == 8 + 7 * 8 and _lib.Lora.rank.offset == 8 and _lib.Lora.ranks.offset == 56
    assert ctypes.sizeof(_lib.LogitCtl) == 11 * 8


def test_no_rows_need_no_row_arrays():
    """An empty batch: its per-row arrays have no elements and may be null, whatever else the controls hold."""
    for kw in (dict(mask_rows=None), dict(spans=None, penalties=None), dict(spans=None), dict(penalties=None)):
        assert _process(M=0, x=None, out=None, token=None, ctl=_ctl(**kw)) == _lib.AIPU_EINVAL
        assert b"null context" in _lib.lib().aipu_last_error()  # the last thing that is checked


@pytest.mark.parametrize("n,text", [(1 << 30, b"penalties need"), ((1 << 30) - 1, b"null context")])
def test_contexts_are_as_long_as_their_counts(n, text):
    """A token's count has 30 bits."""
    assert _process(ctl=_ctl(n_tokens=n)) == _lib.AIPU_EINVAL
    assert text in _lib.lib().aipu_last_error()


@pytest.mark.parametrize("M,text", [(1 << 24, b"too many rows"), ((1 << 24) - 256, b"null context")])
def test_projection_refuses_more_rows_than_its_grid(M, text):
    """65535 tiles of 256 rows."""
    L = _lib.lib()
    assert L.aipu_q4k_gemm_lora(None, 0, 16, 32, 256, 16, M, _lora(), 16, 16, 256, 1 << 50, None) == _lib.AIPU_EINVAL
    assert text in L.aipu_last_error()
