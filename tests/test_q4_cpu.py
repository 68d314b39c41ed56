"""4-bit rows without a GPU: refusals of the C entry points (made before anything is launched) and the 64-bit definition
the GPU tests compare with."""
import ctypes

import pytest
import torch

from tests import q4_util

P16 = ctypes.c_void_p(0x10000)      # 16-byte aligned stand-ins: a refused call never touches them
ODD = ctypes.c_void_p(0x10002)


def _lib():
    from diffcache_b200 import _lib as binding

    return binding.load()


def _refused(rc, lib, text):
    assert rc == -1, rc
    assert text in lib.dc_last_error().decode(), lib.dc_last_error()


def test_engine_calls_refuse_a_null_engine():
    lib = _lib()
    assert lib.dc_store_bits(None) == 0
    assert lib.dc_write_rows(None, P16, P16, 0, 1, 0, 0, 0, 0) == -1
    assert lib.dc_read_rows(None, 0, None, 1, P16, P16, 0) == -1
    assert lib.dc_score_rows(None, P16, 0, 1, P16, 1, 0) == -1
    assert lib.dc_attend_rows(None, P16, 0, None, -1, None, None, None, 0, None, None, 0, 0, 0, 0.0, P16, None, 0) == -1
    assert lib.dc_export_q4(None, P16, P16, P16, P16) == -1
    assert lib.dc_import_q4(None, P16, P16, P16, P16, 1) == -1


def test_create_q4_refuses_what_create_refuses():
    lib, h = _lib(), ctypes.c_void_p()
    _refused(lib.dc_create_q4(1, 30, 8, 128, 1024, 0, 0, ctypes.byref(h)), lib, "multiple")
    _refused(lib.dc_create_q4(1, 32, 8, 96, 1024, 0, 0, ctypes.byref(h)), lib, "head_dim")
    _refused(lib.dc_create_q4(1, 32, 8, 128, 0, 0, 0, ctypes.byref(h)), lib, "max_ctx_len")
    _refused(lib.dc_create_q4(1, 32, 8, 128, 1024, 3, 0, ctypes.byref(h)), lib, "dtype")
    _refused(lib.dc_create_q4(20000, 32, 8, 128, 1024, 0, 0, ctypes.byref(h)), lib, "65535")


WRITE = dict(keys=P16, vals=P16, sb=1024, sh=128, ss=128, n_prob=4, kv_heads=2, n=8, head_dim=128, dtype=0, kc=P16, ks=P16,
             vc=P16, vs=P16, prob_rows=64, row0=0)


@pytest.mark.parametrize("change,text", [
    (dict(keys=None), "null"), (dict(vs=None), "null"), (dict(keys=ODD), "aligned"), (dict(kc=ODD), "aligned"),
    (dict(ss=12), "multiples of 8"), (dict(sb=-1024), "non-negative"), (dict(head_dim=96), "head_dim"), (dict(dtype=2), "dtype"),
    (dict(n=65), "rows"), (dict(row0=57), "rows"), (dict(row0=-1), "rows"), (dict(n=-1), "rows"), (dict(kv_heads=0), "kv_heads"),
    (dict(n_prob=65536), "n_prob"), (dict(prob_rows=1 << 31), "prob_rows"), (dict(row0=1 << 62), "rows"),
])
def test_write_rows_refusals(change, text):
    lib = _lib()
    _refused(lib.dc_q4_write_rows(*{**WRITE, **change}.values(), 0), lib, text)


READ = dict(codes=P16, scales=P16, prob_rows=64, n_rows=64, n_prob=4, head_dim=128, dtype=0, row0=0, ids=None, ids_stride=0,
            n=8, out=P16)


@pytest.mark.parametrize("change,text", [
    (dict(codes=None), "null"), (dict(out=None), "null"), (dict(scales=ODD), "aligned"), (dict(out=ODD), "aligned"),
    (dict(head_dim=32), "head_dim"), (dict(n_rows=65), "n_rows"), (dict(n=-1), "n="), (dict(row0=-1), "row0"),
    (dict(ids=P16, ids_stride=7), "ids_stride"), (dict(n=1 << 31), "n="),
])
def test_read_rows_refusals(change, text):
    lib = _lib()
    _refused(lib.dc_q4_read_rows(*{**READ, **change}.values(), 0), lib, text)


SCAN = dict(codes=P16, scales=P16, prob_rows=64, n_prob=4, n=64, head_dim=128, dtype=0, q=P16, q_mode=0, group=1, scores=P16,
            stride=64, minmax=None)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(scores=None), "null"), (dict(codes=ODD), "aligned"), (dict(q=ODD), "aligned"),
    (dict(n=65), "n="), (dict(stride=63), "score_stride"), (dict(q_mode=2), "q_mode"), (dict(q_mode=1, group=0), "group"),
    (dict(dtype=-1), "dtype"), (dict(head_dim=512), "head_dim"),
])
def test_score_scan_refusals(change, text):
    lib = _lib()
    _refused(lib.dc_q4_score_scan(*{**SCAN, **change}.values(), 0), lib, text)


ATTEND = dict(kc=P16, ks=P16, vc=P16, vs=P16, prob_rows=64, n_rows=64, n_prob=4, kv_heads=2, group=4, head_dim=128, dtype=0,
              q=P16, sel=None, sel_stride=0, n_sel=-1, sel_base=0, lens=None, k_new=None, v_new=None, res_k=None, res_v=None,
              sb=0, sh=0, res_len=0, scale=0.0, out=P16, lse=None, acc=None, ml=None, scratch=P16)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(scratch=None), "null"), (dict(kc=None), "null store"), (dict(n_rows=65), "n_rows"),
    (dict(n_prob=5), "multiple of kv_heads"), (dict(group=0), "group"), (dict(group=65), "group"),
    (dict(n_sel=4), "without ids"), (dict(n_sel=4, sel=P16, sel_stride=3), "sel_stride"),
    (dict(n_sel=4, sel=P16, sel_stride=4, lens=P16), "lens"), (dict(k_new=P16), "both"), (dict(res_k=P16), "both"),
    (dict(res_len=3), "resident"), (dict(res_len=-1), "negative"), (dict(out=None), "either"), (dict(acc=P16, ml=P16), "either"),
    (dict(res_k=P16, res_v=P16, sb=12), "multiples of 8"), (dict(q=ODD), "aligned"), (dict(vs=ODD), "aligned"),
    (dict(k_new=ODD, v_new=P16), "aligned"), (dict(head_dim=80), "head_dim"),
])
def test_attend_refusals(change, text):
    lib = _lib()
    _refused(lib.dc_q4_attend(*{**ATTEND, **change}.values(), 0), lib, text)


def test_empty_problems_are_accepted_without_a_launch():
    lib = _lib()
    assert lib.dc_q4_write_rows(*{**WRITE, "n_prob": 0}.values(), 0) == 0
    assert lib.dc_q4_write_rows(*{**WRITE, "n": 0}.values(), 0) == 0
    assert lib.dc_q4_read_rows(*{**READ, "n": 0}.values(), 0) == 0
    assert lib.dc_q4_score_scan(*{**SCAN, "n": 0, "stride": 0}.values(), 0) == 0
    assert lib.dc_q4_attend(*{**ATTEND, "n_prob": 0}.values(), 0) == 0
    assert lib.dc_q4_attend_scratch_bytes(1, 4, 128) > 0


def test_store_bits_option():
    from diffcache_b200 import DiffCacheGPU

    with pytest.raises(ValueError, match="store_bits"):
        DiffCacheGPU(1, 32, 8, 128, store_bits=8, device=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_definition(dtype):
    """Properties of the definition itself: the error bound, zeros kept, ties to even, the caps at both ends."""
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(50, 128, generator=gen) * torch.logspace(-4, 3, 50)[:, None]).to(dtype)
    c, s = q4_util.quantise(x)
    err = (x.double().reshape(50, 4, 32) - c * s).abs()
    assert (err <= s / 2 + 7 * s * q4_util.HALF_STEP[dtype]).all()
    assert c.abs().max() == 7 and torch.equal(c, c.round())
    assert (q4_util.stored(torch.zeros(1, 64, dtype=dtype)) == 0).all()
    tie = torch.zeros(1, 64, dtype=dtype)
    tie[0, :6] = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5])     # scale 1
    assert q4_util.stored(tie)[0, :6].tolist() == [7.0, 0.0, 2.0, 2.0, 0.0, -2.0]
    big = torch.full((1, 64), torch.finfo(dtype).max, dtype=dtype)
    assert torch.isfinite(q4_util.stored(big).to(dtype)).all()
    bad = torch.ones(1, 64, dtype=dtype)
    bad[0, 3] = float("inf")
    back = q4_util.stored(bad)
    assert torch.isnan(back[0, :32]).all() and (back[0, 32:] == q4_util.stored(torch.ones(1, 64, dtype=dtype))[0, 32:]).all()
