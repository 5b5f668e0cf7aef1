"""Host side of the quantized K/V cache (CPU only: no kernel runs): the C
entry points refuse bad calls before they touch a device, KVRows and
QuantKVCache check what the host knows."""

import ctypes

import pytest
import torch

from qwen_megakernel_b200 import KVCacheError, KVRows, QuantKVCache, cdll
from qwen_megakernel_b200 import kv_cache as kvmod

QMK_ERR_ARGS = 1
QMK_ERR_WORKSPACE = 6

vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


class Cache(ctypes.Structure):
    _fields_ = [("k_codes", vp), ("v_codes", vp), ("k_scales", vp), ("v_scales", vp), ("code_seq_stride", i64),
                ("scale_seq_stride", i64), ("num_seqs", i32), ("num_kv_heads", i32), ("head_dim", i32), ("bits", i32),
                ("capacity", i32), ("max_seq_len", i32)]


class Rows(ctypes.Structure):
    _fields_ = [("rows", i32), ("segments", i32), ("max_rows", i32), ("start", vp), ("row_offsets", vp), ("seq", vp)]


class Tensor(ctypes.Structure):
    _fields_ = [("data", vp), ("dtype", i32), ("row_stride", i64), ("head_stride", i64)]


FAKE = 1 << 20  # an aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    lib = cdll()
    P = ctypes.POINTER
    lib.qmk_kv_write.argtypes = [P(Cache), P(Rows), P(Tensor), P(Tensor), vp, vp]
    lib.qmk_kv_read.argtypes = [P(Cache), P(Rows), P(Tensor), P(Tensor), vp, vp]
    lib.qmk_kv_attend.argtypes = [P(Cache), P(Rows), P(Tensor), i32, P(Tensor), ctypes.c_float, vp, ctypes.c_size_t,
                                  vp, vp]
    lib.qmk_kv_attend_workspace_bytes.argtypes = [P(Cache), P(Rows), i32, i32]
    lib.qmk_kv_attend_workspace_bytes.restype = ctypes.c_size_t
    lib.qmk_get_last_error_message.restype = ctypes.c_char_p
    return lib


def _cache(**kw):
    f = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, code_seq_stride=8 * 256 * 64,
             scale_seq_stride=8 * 256 * 4, num_seqs=2, num_kv_heads=8, head_dim=128, bits=4, capacity=256,
             max_seq_len=200)
    f.update(kw)
    return Cache(**f)


def _rows(**kw):
    f = dict(rows=3, segments=3, max_rows=1, start=FAKE, row_offsets=None, seq=None)
    f.update(kw)
    return Rows(**f)


def _tensor(**kw):
    f = dict(data=FAKE, dtype=0, row_stride=1024, head_stride=128)
    f.update(kw)
    return Tensor(**f)


BAD_CACHES = [dict(k_codes=None), dict(v_scales=None), dict(bits=3), dict(head_dim=96), dict(num_seqs=0),
              dict(num_kv_heads=0), dict(max_seq_len=0), dict(max_seq_len=257), dict(capacity=200, max_seq_len=200),
              dict(code_seq_stride=1024), dict(scale_seq_stride=1024), dict(code_seq_stride=8 * 256 * 64 + 8),
              dict(scale_seq_stride=8 * 256 * 4 + 4), dict(k_codes=FAKE + 8), dict(v_scales=FAKE + 2)]
BAD_ROWS = [dict(rows=-1), dict(segments=-1), dict(max_rows=-1), dict(start=None), dict(rows=4), dict(max_rows=257)]
BAD_TENSORS = [dict(data=None), dict(dtype=3), dict(dtype=-1), dict(data=FAKE + 1)]


@pytest.mark.parametrize("what", BAD_CACHES, ids=str)
def test_c_entries_refuse_bad_caches(lib, what):
    c, r, t = _cache(**what), _rows(), _tensor()
    assert lib.qmk_kv_write(c, r, t, t, None, None) == QMK_ERR_ARGS
    assert b"qmk_kv_write" in lib.qmk_get_last_error_message()
    assert lib.qmk_kv_read(c, r, t, t, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_attend(c, r, t, 16, t, 1.0, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_attend_workspace_bytes(c, r, 16, 0) == 0


@pytest.mark.parametrize("what", BAD_ROWS, ids=str)
def test_c_entries_refuse_bad_rows(lib, what):
    c, r, t = _cache(), _rows(**what), _tensor()
    assert lib.qmk_kv_write(c, r, t, t, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_read(c, r, t, t, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_attend(c, r, t, 16, t, 1.0, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_attend_workspace_bytes(c, r, 16, 0) == 0


@pytest.mark.parametrize("what", BAD_TENSORS, ids=str)
def test_c_entries_refuse_bad_tensors(lib, what):
    c, r, t, bad = _cache(), _rows(), _tensor(), _tensor(**what)
    for k, v in ((bad, t), (t, bad)):
        assert lib.qmk_kv_write(c, r, k, v, None, None) == QMK_ERR_ARGS
        assert lib.qmk_kv_read(c, r, k, v, None, None) == QMK_ERR_ARGS
        assert lib.qmk_kv_attend(c, r, k, 16, v, 1.0, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS


def test_c_entries_refuse_mixed_types_heads_and_workspaces(lib):
    c, r, t, h = _cache(), _rows(), _tensor(), _tensor(dtype=1)
    assert lib.qmk_kv_write(c, r, t, h, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_read(c, r, t, h, None, None) == QMK_ERR_ARGS
    assert lib.qmk_kv_attend(c, r, t, 16, h, 1.0, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS
    for heads in (0, -8, 4, 12, 8 * 17):
        assert lib.qmk_kv_attend(c, r, t, heads, t, 1.0, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS
        assert lib.qmk_kv_attend_workspace_bytes(c, r, heads, 0) == 0
    assert lib.qmk_kv_attend_workspace_bytes(c, r, 16, 7) == 0
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert lib.qmk_kv_attend(c, r, t, 16, t, scale, FAKE, 1 << 30, None, None) == QMK_ERR_ARGS
    need = lib.qmk_kv_attend_workspace_bytes(c, r, 16, 0)
    assert need > 0 and need % 256 == 0
    for ws, n in ((None, need), (FAKE, need - 1), (FAKE + 128, need)):
        assert lib.qmk_kv_attend(c, r, t, 16, t, 1.0, ws, n, None, None) == QMK_ERR_WORKSPACE


def test_no_rows_is_no_work(lib):
    """A call of no rows returns without a launch (there is no device here)."""
    c, t = _cache(), _tensor()
    for r in (_rows(rows=0, segments=0, start=None), _rows(rows=0, segments=3, row_offsets=FAKE)):
        assert lib.qmk_kv_write(c, r, t, t, None, None) == 0
        assert lib.qmk_kv_read(c, r, t, t, None, None) == 0
        assert lib.qmk_kv_attend(c, r, t, 16, t, 1.0, None, 0, None, None) == 0


def test_status_bits_match_the_header():
    import os
    import re

    from conftest import ROOT

    src = open(os.path.join(ROOT, "include", "qwen_megakernel.h")).read()
    for name in ("BAD_ROW", "NONFINITE", "TIMEOUT", "COPIES_PENDING", "GROUP", "CAPACITY_STEP", "MAX_RATIO"):
        value = int(re.search(rf"#define QMK_KV_{name} (\d+)", src).group(1))
        assert getattr(kvmod, name) == value, name


def test_rows_segments():
    r = KVRows([5, 0, 7], [2, 0, 3], [1, 0, 1], device="cpu")
    assert r.rows == 5 and r.max_rows == 3
    assert r.row_offsets.tolist() == [0, 2, 2, 5] and r.start.tolist() == [5, 0, 7] and r.seq.tolist() == [1, 0, 1]
    one = KVRows([4, 9], device="cpu")
    assert one.rows == 2 and one.max_rows == 1 and one.row_offsets is None and one.seq is None
    t = torch.zeros(3, dtype=torch.int32)
    assert KVRows.from_tensors(t).rows == 3
    assert KVRows.from_tensors(t, torch.zeros(4, dtype=torch.int32), rows=9, max_rows=4).max_rows == 4


@pytest.mark.parametrize("args", [([],), ([-1],), ([0], [-1]), ([0], [1, 2]), ([0, 1], None, [0]), ([2**31],),
                                  ([0, 0], [2**30, 2**30])], ids=str)
def test_rows_refuse(args):
    with pytest.raises(ValueError):
        KVRows(*args, device="cpu")


def test_rows_from_tensors_refuse():
    t = torch.zeros(3, dtype=torch.int32)
    for kw in (dict(rows=4), dict(max_rows=2), dict(row_offsets=t), dict(row_offsets=t, rows=3),
               dict(row_offsets=t, rows=-1, max_rows=1)):
        with pytest.raises(ValueError):
            KVRows.from_tensors(t, **kw)


@pytest.mark.parametrize("kw", [dict(bits=5), dict(head_dim=32), dict(num_seqs=0), dict(max_seq_len=0),
                                dict(num_layers=0), dict(num_kv_heads=0)], ids=str)
def test_cache_refuses(kw):
    args = dict(num_seqs=1, max_seq_len=10, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError):
        QuantKVCache(**args)


def test_cache_checks_what_the_host_knows():
    c = QuantKVCache(2, 200, num_layers=3, num_kv_heads=2, head_dim=64, bits=4, device="cpu")
    assert c.capacity == 256 and c.k_codes.shape == (2, 3, 2, 256, 32) and c.v_scales.shape == (2, 3, 2, 256, 2)
    assert c.nbytes == 2 * (2 * 3 * 2 * 256) * (32 + 4)
    x = torch.zeros(2, 2, 64)

    def refused(rows, k=x, layer=0):
        with pytest.raises(ValueError):
            c.write(k, k, rows, layer)
        with pytest.raises(ValueError):
            c.read(rows, layer, out=(k, k))
        with pytest.raises(ValueError):
            c.attend(k, rows, layer)

    refused(KVRows([199], [2], device="cpu"))  # past max_seq_len, though inside the capacity
    refused(KVRows([0, 0], seq_ids=[0, 2], device="cpu"))
    refused(KVRows([0], [3], device="cpu"))  # 3 rows for 2
    refused(KVRows([0, 0], device="cpu"), layer=3)
    refused(KVRows([0, 0], device="cpu"), layer=-1)
    refused(KVRows([0, 0], device="cpu"), k=torch.zeros(2, 2, 128))
    refused(KVRows([0, 0], device="cpu"), k=torch.zeros(2, 128))
    t = torch.zeros(2, dtype=torch.int32)
    refused(KVRows.from_tensors(t, torch.zeros(3, dtype=torch.int32), rows=2, max_rows=201))
    with pytest.raises(ValueError):  # one position twice
        c.write(x, x, KVRows([4, 4], None, [1, 1], device="cpu"))
    for heads in (1, 3, 34):
        with pytest.raises(ValueError):
            c.attend(torch.zeros(2, heads, 64), KVRows([0, 0], device="cpu"))
    with pytest.raises(ValueError):
        c.attend(x, KVRows([0, 0], device="cpu"), out=torch.zeros(2, 2, 64, dtype=torch.bfloat16))


def test_no_cpu_path():
    """There is no CPU kernel: the operators are registered for CUDA only."""
    c = QuantKVCache(1, 8, num_kv_heads=1, head_dim=64, device="cpu")
    with pytest.raises(NotImplementedError):
        c.write(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), KVRows([0], device="cpu"))


def test_check_status_names_the_findings():
    c = QuantKVCache(1, 8, num_kv_heads=1, head_dim=64, device="cpu")
    c.check_status()
    c.status.fill_(kvmod.BAD_ROW | kvmod.NONFINITE)
    with pytest.raises(KVCacheError, match="out of range.*NaN or infinity"):
        c.check_status()
    c.check_status()


def test_batch_forward_kvq_refuses(lib):
    """The forward pass over a quantized cache checks its arguments before it
    touches a device."""
    from test_batch_host import QmkBatchArgs

    class Kvq(ctypes.Structure):
        _fields_ = [("cache", Cache), ("code_layer_stride", i64), ("scale_layer_stride", i64), ("rows", Rows),
                    ("workspace", vp), ("workspace_bytes", ctypes.c_size_t), ("status", vp)]

    P = ctypes.POINTER
    lib.qmk_batch_forward_kvq.argtypes = [P(QmkBatchArgs), P(Kvq), vp]
    lib.qmk_batch_workspace_bytes.restype = ctypes.c_size_t
    ptrs = (vp * 22)(*([FAKE] * 22))
    rows = _rows()
    need = lib.qmk_kv_attend_workspace_bytes(_cache(), rows, 16, 1)

    def call(cache=None, rows=rows, code=8 * 256 * 64, scale=8 * 256 * 4, ws=FAKE, n=need, **kw):
        f = dict(embed_weight=FAKE, layer_ptrs=ctypes.cast(ptrs, vp).value, final_norm_weight=FAKE,
                 lm_head_weight=FAKE, cos_table=FAKE, sin_table=FAKE, num_seqs=2, num_layers=2, max_seq_len=200,
                 num_rows=3, tokens=FAKE, row_seq=FAKE, row_pos=FAKE, workspace=FAKE, workspace_bytes=0)
        f.update(kw)
        return lib.qmk_batch_forward_kvq(QmkBatchArgs(**f), Kvq(cache or _cache(), code, scale, rows, ws, n, None),
                                         None)

    assert lib.qmk_batch_forward_kvq(QmkBatchArgs(), None, None) == QMK_ERR_ARGS
    assert call() == QMK_ERR_WORKSPACE  # everything but the (empty) batch workspace is in order
    assert b"qmk_batch_forward:" in lib.qmk_get_last_error_message()
    for what in BAD_CACHES:
        assert call(cache=_cache(**what)) == QMK_ERR_ARGS
    for bad in (dict(cache=_cache(num_kv_heads=4)), dict(cache=_cache(head_dim=64)), dict(num_seqs=1),
                dict(max_seq_len=199), dict(num_rows=4), dict(rows=_rows(segments=0, rows=3, row_offsets=FAKE)),
                dict(rows=_rows(max_rows=0)), dict(code=1024), dict(scale=1024), dict(code=8 * 256 * 64 + 8),
                dict(scale=8 * 256 * 4 + 4), dict(tokens=None), dict(num_layers=0)):
        assert call(**bad) == QMK_ERR_ARGS, bad
    for bad in (dict(ws=None), dict(n=need - 1), dict(ws=FAKE + 128)):
        assert call(**bad) == QMK_ERR_WORKSPACE, bad
        assert b"kvq" in lib.qmk_get_last_error_message()
