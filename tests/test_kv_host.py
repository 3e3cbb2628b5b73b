"""Paged KV-cache checks on the CPU (no GPU): refusals, extents, visible spans, bad lengths, the
binding's structures, and what the Python layer refuses before the library is called."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import gfd_b200
from gfd_b200 import GFD_ERR_INVALID, kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_VP = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    out = os.path.join(tempfile.mkdtemp(prefix="gfdt_"), "libgfdtkv.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-Wall", "-Werror",
                           "-I", os.path.join(ROOT, "gfd_b200", "csrc"), "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "kv_logic.cpp"), "-o", out])
    l = ctypes.CDLL(out)
    u64p = ctypes.POINTER(ctypes.c_uint64)
    for name, args in {"cache": [_VP, ctypes.c_int, u64p], "batch": [_VP, _VP, ctypes.c_int64], "append": [_VP, _VP],
                       "attend": [_VP, _VP], "merge": [_VP],
                       "rows": [_VP, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int,
                                u64p]}.items():
        f = getattr(l, "gfdt_kv_" + name)
        f.argtypes, f.restype = args, ctypes.c_char_p
    l.gfdt_kv_span.argtypes = [ctypes.c_int32] * 4 + [ctypes.c_int, _VP]
    l.gfdt_kv_seq.argtypes = [ctypes.c_int32] * 3 + [ctypes.c_int64, ctypes.c_int32, _VP]
    return l


def cache(**kw):
    c = kv._Cache(k=1 << 20, v=(1 << 20) + 4096, blocks=10, block_stride=2 * 16 * 8 * 128, token_stride=8 * 128,
                  head_stride=128, block_tokens=16, heads=8, head_dim=128, dtype=kv.BF16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_layout_matches_header(lib):
    v = (ctypes.c_uint64 * 12)()
    lib.gfdt_kv_layout(v)
    want = []
    for s, last in ((kv._Cache, "dtype"), (kv._Batch, "table_width"), (kv._Rows, "head_stride"), (kv._Append, "interleaved"),
                    (kv._Attend, "softcap"), (kv._Merge, "out_dtype")):
        want += [ctypes.sizeof(s), getattr(s, last).offset]
    assert list(v) == want


def test_constants_match_header():
    import re
    hdr = open(os.path.join(ROOT, "include", "gfd_b200.h")).read()
    for name, value in re.findall(r"#define GFD_KV_(\w+) (\d+)u?", hdr):
        assert getattr(kv, name) == int(value), name
    for name in ("BF16", "FP16", "FP32"):
        assert f"GFD_{name} = {getattr(kv, name)}" in hdr


def test_cache_checks(lib):
    n = ctypes.c_uint64()

    def check(write=1, **kw):
        c = cache(**kw)
        return lib.gfdt_kv_cache(ctypes.byref(c), write, ctypes.byref(n))

    assert check() is None and n.value == 2 * (9 * 32768 + 15 * 1024 + 7 * 128 + 128)
    for kw in (dict(dtype=kv.FP32), dict(dtype=9), dict(head_dim=96), dict(head_dim=0), dict(heads=0), dict(heads=1025),
               dict(block_tokens=8), dict(block_tokens=24), dict(block_tokens=0), dict(block_tokens=2048), dict(blocks=0),
               dict(blocks=1 << 31), dict(k=None), dict(v=None), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2),
               dict(token_stride=1020), dict(token_stride=-1024), dict(head_stride=0), dict(head_stride=64),
               dict(token_stride=0), dict(block_stride=15 * 1024), dict(block_stride=1 << 38), dict(v=1 << 20)):
        assert check(**kw) is not None, kw
    assert check(write=0, v=1 << 20) is None                     # reading K as V is fine
    assert check(blocks=1, block_stride=0) is None               # strides of single things are not used
    assert check(heads=1, head_stride=-3) is None
    assert check(token_stride=128, head_stride=16 * 128) is None  # heads outside tokens
    assert check(blocks=(1 << 31) - 1, block_stride=(1 << 38) - 8) is not None  # 2^70 bytes


def test_batch_checks(lib):
    def check(shared=0, **kw):
        b = kv._Batch(row_start=64, kv_len=128, table=256, table_stride=5, rows=7, seqs=3, table_width=5)
        for k, v in kw.items():
            setattr(b, k, v)
        c = cache()
        return lib.gfdt_kv_batch(ctypes.byref(b), ctypes.byref(c), shared)

    assert check() is None
    assert check(rows=0, row_start=None) is None and check(seqs=0, table=None) is None
    assert check(table_width=0, table=None, table_stride=0) is None
    for kw in (dict(rows=-1), dict(rows=1 << 30), dict(seqs=-1), dict(seqs=4097), dict(table_width=-1), dict(table_stride=4),
               dict(table_stride=-5), dict(row_start=None), dict(kv_len=None), dict(table=None), dict(row_start=66),
               dict(kv_len=129), dict(table=257), dict(table_width=1 << 27, table_stride=1 << 27), dict(shared=-1),
               dict(shared=1 << 30)):
        assert check(**kw) is not None, kw
    assert check(seqs=1, table_stride=0) is None


def test_rows_checks(lib):
    n = ctypes.c_uint64()

    def check(rows, heads, row_stride, head_stride, data=4096, dim=64, dtype=kv.BF16, out=0):
        r = kv._Rows(data, row_stride, head_stride)
        return lib.gfdt_kv_rows(ctypes.byref(r), rows, heads, dim, dtype, out, ctypes.byref(n))

    assert check(5, 4, 256, 64) is None and n.value == 2 * (4 * 256 + 3 * 64 + 64)
    assert check(5, 4, 256, 64, dtype=kv.FP32) is None and n.value == 4 * 1280
    assert check(5, 4, 256, 0) is None              # a head broadcast: read
    assert check(5, 4, 256, 0, out=1) is not None   # but not written
    assert check(5, 4, 64, 5 * 64, out=1) is None   # heads outermost
    assert check(5, 4, 64, 4 * 64, out=1) is not None
    assert check(1, 1, -7, 3, out=1) is None        # strides of single things are not used
    for args in ((5, 4, 255, 64), (5, 4, 256, 60), (5, 4, -256, 64), (1 << 29, 8192, 1 << 50, 64)):
        assert check(*args) is not None, args
    assert check(5, 4, 256, 64, data=None) is not None and check(5, 4, 256, 64, data=4104) is not None


def test_operator_argument_checks(lib):
    c = cache()

    def attend(**kw):
        a = kv._Attend(q=kv._Rows(4096, 4096, 128), out=kv._Rows(8192, 4096, 128), q_heads=32, out_dtype=kv.BF16, causal=1,
                       scale=0.1)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gfdt_kv_attend(ctypes.byref(a), ctypes.byref(c))

    assert attend() is None and attend(out_dtype=kv.FP32) is None and attend(q_heads=8) is None
    for kw in (dict(q_heads=0), dict(q_heads=12), dict(q_heads=-8), dict(q_heads=16384), dict(out_dtype=kv.FP16), dict(out_dtype=3),
               dict(max_q_len=-1), dict(window=-1), dict(window=(1 << 30) + 1), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(softcap=-0.5), dict(softcap=float("nan")), dict(lse=2), dict(alibi=6), dict(prefix_len=1), dict(status=3),
               dict(out=kv._Rows(4096, 4096, 128))):
        assert attend(**kw) is not None, kw

    def append(**kw):
        a = kv._Append(q_heads=32, rot_dim=128, inv_freq=64)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gfdt_kv_append(ctypes.byref(a), ctypes.byref(c))

    assert append() is None and append(rot_dim=0, inv_freq=None) is None and append(q_heads=0) is None
    for kw in (dict(rot_dim=-16), dict(rot_dim=8), dict(rot_dim=144), dict(inv_freq=None), dict(inv_freq=2), dict(q_heads=-1),
               dict(positions=3), dict(status=2), dict(q=kv._Rows(16, 8, 8), q_out=kv._Rows(16, 16, 8))):
        assert append(**kw) is not None, kw

    def merge(**kw):
        a = kv._Merge(parts=kv._Rows(4096, 512, 128), part_stride=5120, part_lse=64, out=kv._Rows(1 << 20, 512, 128), rows=10,
                      part_count=3, heads=4, head_dim=128, part_dtype=kv.FP32, out_dtype=kv.BF16)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gfdt_kv_merge(ctypes.byref(a))

    assert merge() is None and merge(rows=0, part_lse=None) is None
    for kw in (dict(part_count=0), dict(part_count=1025), dict(heads=0), dict(head_dim=80), dict(part_dtype=5), dict(out_dtype=-1),
               dict(part_stride=-8), dict(part_stride=12), dict(part_lse=None), dict(part_lse=3), dict(lse=1), dict(rows=-1),
               dict(out=kv._Rows(4096 + 2 * 5120 * 4, 512, 128))):
        assert merge(**kw) is not None, kw


def test_spans_match_the_mask(lib):
    """[0, pre) and [lo, hi) are disjoint and name exactly the keys the mask lets through."""
    out = (ctypes.c_int32 * 3)()
    rng = np.random.default_rng(1)
    for _ in range(3000):
        n = int(rng.integers(1, 40))
        p = int(rng.integers(0, n))
        prefix, window, causal = int(rng.integers(-2, 45)), int(rng.integers(0, 12)), int(rng.integers(0, 2))
        lib.gfdt_kv_span(p, n, prefix, window, causal, out)
        pre, lo, hi = out
        want = {j for j in range(n) if j < prefix or ((not causal or j <= p) and (window == 0 or j > p - window))}
        assert 0 <= pre <= lo <= hi <= n
        assert set(range(pre)) | set(range(lo, hi)) == want
    lib.gfdt_kv_span((1 << 30) - 1, 1 << 30, 0, 1 << 30, 1, out)
    assert list(out) == [0, 0, 1 << 30]


def test_bad_lengths(lib):
    out = (ctypes.c_int32 * 3)()
    assert lib.gfdt_kv_seq(3, 5, 2, 16, 0, out) == 1 and list(out) == [3, 2, 2]
    assert lib.gfdt_kv_seq(3, 5, 16, 16, 2, out) == 1
    for args in ((3, 5, 1, 16, 0), (3, 5, 17, 16, 0), (3, 5, -1, 16, 0), (3, 6, 10, 16, 2)):
        assert lib.gfdt_kv_seq(*args, out) == 0, args
    for n in (-5, 0, 100):  # a sequence without rows has nothing to skip
        assert lib.gfdt_kv_seq(5, 5, n, 16, 1, out) == 1 and list(out) == [5, 0, 0]


def test_entry_points_refuse_null_context():
    l = gfd_b200.load()
    assert l.gfd_kv_append(None, None, None, None, None) == GFD_ERR_INVALID
    assert l.gfd_kv_attend(None, None, None, None, None) == GFD_ERR_INVALID
    assert l.gfd_kv_attend_shared(None, None, None, None, 0, None, None) == GFD_ERR_INVALID
    assert l.gfd_kv_attend_workspace(None, None, None, None, 0, None) == GFD_ERR_INVALID
    assert l.gfd_kv_merge(None, None, None) == GFD_ERR_INVALID


def test_python_layer_refuses_wrong_arrays():
    import torch
    z = torch.zeros
    pool = z(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    for k, v in ((pool[:, 0], z(4, 16, 2, 64, dtype=torch.bfloat16)),               # other strides
                 (pool[:, 0], pool[:3, 1]), (pool[:, 0], pool[:, 1].half()),
                 (pool[:, 0].transpose(2, 3), pool[:, 1].transpose(2, 3)), (z(4, 16, 2, 64), z(4, 16, 2, 64, dtype=torch.float64)),
                 (z(4, 16, 2, 64, dtype=torch.int16), z(4, 16, 2, 64, dtype=torch.int16))):
        with pytest.raises(ValueError):
            kv.PagedCache(None, k, v)
    i = torch.int32
    starts, lens, table = z(3, dtype=i), z(2, dtype=i), z(2, 4, dtype=i)
    for args in ((starts[:2], lens, table), (starts.long(), lens, table), (starts, lens.float(), table), (starts, lens, table.long()),
                 (starts, lens, table[:1]), (starts, lens, table.t().contiguous().t()), (z(6, dtype=i)[::2], lens, table)):
        with pytest.raises(ValueError):
            kv.Batch(*args)
    c, b = kv.PagedCache(None, pool[:, 0], pool[:, 1]), kv.Batch(starts, lens, table)
    q, out = z(5, 4, 64, dtype=torch.bfloat16), z(5, 4, 64, dtype=torch.bfloat16)
    for args, kw in (((q.half(), out), {}), ((q, out[:4]), {}), ((q, out.double()), {}), ((q[:, :, ::2], out), {}),
                     ((q, out), dict(lse=z(4, 5))), ((q, out), dict(alibi=z(3))), ((q, out), dict(prefix_len=z(2))),
                     ((q, out), dict(status=z(1)))):
        with pytest.raises(ValueError):
            c.attend(b, *args, **kw)
    with pytest.raises(ValueError):
        c.attend_shared(b, z(1, dtype=i), 17, q, out)
    k = z(5, 2, 64, dtype=torch.bfloat16)
    for args, kw in (((k, k[:4]), {}), ((k, k.half()), {}), ((k, k), dict(q=q)), ((k, k), dict(q=q, q_out=out[:4])),
                     ((k, k), dict(positions=z(5))), ((k, k), dict(inv_freq=z(16, dtype=torch.float64)))):
        with pytest.raises(ValueError):
            c.append(b, *args, **kw)
    with pytest.raises(ValueError):
        kv.merge(None, z(2, 3, 4, 64), z(2, 3, 5), z(3, 4, 64))
    with pytest.raises(ValueError):
        c.fetch(0, [0, 1], [0])
    with pytest.raises(ValueError):
        c.fetch(0, [0], [4])


def test_block_entries():
    """fetch and offload name K and V of each block with the bytes of its tokens."""
    import torch
    pool = torch.zeros(6, 2, 16, 2, 64, dtype=torch.float16)
    c = kv.PagedCache(None, pool[:, 0], pool[:, 1])
    half = 16 * 2 * 64 * 2
    e = c._block_entries(1 << 30, [3, 0], [1, 5], False)
    base = pool.data_ptr()
    assert e["dst"].tolist() == [base + 2 * half, base + 3 * half, base + 10 * half, base + 11 * half]
    assert e["src"].tolist() == [(1 << 30) + 6 * half, (1 << 30) + 7 * half, 1 << 30, (1 << 30) + half]
    assert e["size"].tolist() == [half] * 4
    r = c._block_entries(1 << 30, [3, 0], [1, 5], True)
    assert r["dst"].tolist() == e["src"].tolist() and r["src"].tolist() == e["dst"].tolist()
    apart = torch.zeros(2, 6, 2, 16, 64, dtype=torch.float16)  # heads outside tokens
    c = kv.PagedCache(None, apart[0].transpose(1, 2), apart[1].transpose(1, 2))
    with pytest.raises(ValueError):
        c.fetch(0, [0], [0])


def test_tiles_hold_every_visible_key_and_no_other(lib):
    """Against a walk over keys: tiles with a key of [0, pre) or of [lo, hi), each once, in order."""
    rng = np.random.default_rng(5)
    lib.gfdt_kv_tiles.argtypes = [_VP, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, _VP]
    cases = [(0, 0, 0, 0, 0), (0, 0, 1, 0, 1), (5, 5, 5, 0, 9), (3, 700, 701, 0, 701), (16, 16, 32, 16, 16), (900, 900, 900, 128, 400)]
    for _ in range(400):
        pre, lo, n = sorted(rng.integers(0, 700, 3).tolist())
        cases.append((pre, lo, int(rng.integers(lo, 701)), int(rng.integers(0, 300)), int(rng.integers(0, 500))))
    for pre, lo, hi, base, length in cases:
        for size in (16, 128):
            span, out = (ctypes.c_int32 * 3)(pre, lo, hi), (ctypes.c_int32 * 3)()
            lib.gfdt_kv_tiles(span, base, length, size, out)
            npre, first, count = out
            got = [i if i < npre else i - npre + first for i in range(count)]
            keys = [j - base for j in range(base, base + length) if j < pre or lo <= j < hi]
            assert got == sorted({j // size for j in keys}), (pre, lo, hi, base, length, size)


def test_cuts_share_the_line_evenly(lib):
    lib.gfdt_kv_cuts.argtypes = [ctypes.c_int64, ctypes.c_uint32, _VP]
    lib.gfdt_kv_last_before.argtypes = [ctypes.c_int64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int64]
    lib.gfdt_kv_last_before.restype = ctypes.c_uint32
    lib.gfdt_kv_div.argtypes, lib.gfdt_kv_div.restype = [ctypes.c_int64] * 2, ctypes.c_int64
    rng = np.random.default_rng(6)
    at = (ctypes.c_int64 * 2049)()
    assert lib.gfdt_kv_cuts(0, 148, at) == 0
    for total, most in [(1, 148), (147, 148), (148, 148), (149, 148), (2 ** 40 + 7, 1776), (2 ** 31, 2048), (2 ** 33 - 1, 1184)] + \
            [(int(rng.integers(1, 5000)), int(rng.integers(1, 2048))) for _ in range(200)]:
        n = lib.gfdt_kv_cuts(total, most, at)
        a = list(at[:n + 1])
        sizes = np.diff(a)
        assert n == min(total, most) and a[0] == 0 and a[n] == total and sizes.min() >= 1 and sizes.max() - sizes.min() <= 1
        for c in {0, n // 3, n - 1}:
            for end in {a[c] + 1, a[c + 1], a[c + 1] + 1, total, (a[c] + total) // 2 + 1}:
                want = max(i for i in range(n) if i == c or (i > c and a[i] < end))
                assert lib.gfdt_kv_last_before(total, most, c, end) == want, (total, most, c, end)
    for a, b in ((0, 1), (2 ** 32 - 1, 1), (2 ** 32, 3), (2 ** 40 + 1, 2 ** 33), (17, 2 ** 34), (2 ** 62, 7), (2 ** 32 - 1, 2 ** 32 - 1)):
        assert lib.gfdt_kv_div(a, b) == a // b


def test_reciprocals_divide_exactly():
    """The kernels divide packed rows by the group, and pages by a block's, with a multiplication: the
    same magic numbers and shifts, at the quotients' edges."""
    for group in list(range(1, 130)) + [255, 256, 1000, 4095, 8191, 8192]:
        magic = -(-2 ** 44 // group)
        for k in (1, 2, 1000, (2 ** 31 - 1) // group):
            for n in (k * group - 1, k * group, k * group + group - 1):
                if 0 <= n < 2 ** 31:
                    assert (n << 20) * magic >> 64 == n // group
    for pages in range(1, 65):
        magic = -(-2 ** 32 // pages)
        for k in (1, 77, (2 ** 26 - 1) // pages):
            for n in (k * pages - 1, k * pages, k * pages + pages - 1):
                if 0 <= n < 2 ** 26:
                    assert n * magic >> 32 == n // pages


def test_attend_parameters_out_of_range(lib):
    c = cache()

    def check(**kw):
        a = kv._Attend(q_heads=32, scale=0.1, out_dtype=kv.BF16)
        a.q.data, a.out.data = 1 << 24, 1 << 25
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gfdt_kv_attend(ctypes.byref(a), ctypes.byref(c))
    assert check() is None and check(softcap=30.0) is None and check(scale=0.0) is None and check(scale=-1.0) is None
    no_rows = kv._Attend(q_heads=32, scale=0.1, out_dtype=kv.BF16)  # whose tensors have no address
    assert lib.gfdt_kv_attend(ctypes.byref(no_rows), ctypes.byref(c)) is None
    for kw in (dict(q_heads=0), dict(q_heads=12), dict(q_heads=8 * 1024 + 8), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(window=-1), dict(max_q_len=-1)):
        assert check(**kw) is not None, kw


def test_table_extent(lib):
    """The table's bytes are counted without wrapping: what is checked is what the kernels read."""
    lib.gfdt_kv_table_bytes.argtypes, lib.gfdt_kv_table_bytes.restype = [_VP], ctypes.c_uint64
    c = cache()

    def check(seqs, width, stride):
        b = kv._Batch(row_start=64, kv_len=128, table=256, table_stride=stride, rows=7, seqs=seqs, table_width=width)
        return lib.gfdt_kv_batch(ctypes.byref(b), ctypes.byref(c), 0), lib.gfdt_kv_table_bytes(ctypes.byref(b))

    for seqs, width, stride in ((1, 5, 0), (1, 5, 1 << 62), (3, 5, 5), (3, 5, 9), (4096, 1000, 1 << 20), (2, 1, (1 << 60) - 2)):
        why, n = check(seqs, width, stride)
        assert why is None and n == 4 * ((seqs - 1) * (stride if seqs > 1 else 0) + width), (seqs, width, stride)
    for seqs, width, stride in ((5, 5, 1 << 62), (2, 5, 1 << 62), (2, 1, 1 << 60), (4096, 1, 1 << 51), (3, 7, (1 << 63) - 1)):
        assert check(seqs, width, stride)[0] is not None, (seqs, width, stride)
    assert check(3, 0, 1 << 62) == (None, 0)  # a table of no width is not read


def test_workspace_of_a_larger_batch_holds_a_smaller_one(lib):
    """Room asked for once, for the largest batch, serves every smaller one, whichever kernels that takes."""
    f = lib.gfdt_kv_workspace
    f.argtypes = [_VP, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int64, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    f.restype = ctypes.c_uint64
    k = ctypes.c_int()

    def room(rows, seqs, max_q, shared=0, heads=8, group=4, d=128):
        c = cache(heads=heads, head_dim=d)
        return f(ctypes.byref(c), rows, seqs, heads * group, max_q, shared, 148, ctypes.byref(k))

    assert room(32768, 4, 8192) >= room(10000, 4, 8192)  # four whole prompts, then prompts among decode steps
    assert k.value == 3 and room(32768, 4, 8192) and k.value == 2 and room(4, 4, 1) and k.value == 1
    rng = np.random.default_rng(8)
    for _ in range(3000):
        group, d = int(rng.choice([1, 3, 4, 8, 16, 17, 40])), int(rng.choice([64, 128]))
        rows, seqs = int(rng.integers(1, 40000)), int(rng.integers(1, 300))
        max_q, shared = int(rng.choice([0, 1, 4, 16, 300, 50000])), int(rng.choice([0, 1, 5000]))
        less = dict(rows=int(rng.integers(1, rows + 1)), seqs=int(rng.integers(1, seqs + 1)), shared=int(rng.integers(0, shared + 1)),
                    max_q=int(rng.integers(0, 60000)) if max_q == 0 else int(rng.integers(1, max_q + 1)))
        assert room(rows, seqs, max_q, shared, group=group, d=d) >= room(**less, group=group, d=d), (rows, seqs, max_q, shared, less)
    assert room(0, 4, 1) == 0 and room(5, 0, 1) == 0


def test_workspace_of_shapes_out_of_range_is_refused(lib):
    f = lib.gfdt_kv_check_workspace
    f.argtypes, f.restype = [_VP, _VP, _VP, ctypes.c_int64], ctypes.c_char_p
    c = cache()

    def check(rows=100, seqs=4, q_heads=32, max_q=9, shared=0):
        b, a = kv._Batch(rows=rows, seqs=seqs), kv._Attend(q_heads=q_heads, max_q_len=max_q)
        return f(ctypes.byref(c), ctypes.byref(b), ctypes.byref(a), shared)

    assert check() is None and check(rows=0, seqs=0) is None and check(rows=(1 << 30) - 1, shared=1 << 30, q_heads=8192) is None
    for kw in (dict(rows=-1), dict(rows=1 << 30), dict(rows=1 << 62), dict(seqs=-1), dict(seqs=4097), dict(q_heads=0), dict(q_heads=12),
               dict(q_heads=8200), dict(q_heads=1 << 30), dict(max_q=-1), dict(shared=-1), dict(shared=(1 << 30) + 1)):
        assert check(**kw) is not None, kw


def test_fetch_refuses_ids_that_are_no_blocks():
    import torch
    pool = torch.zeros(6, 2, 16, 2, 64, dtype=torch.float16)
    c = kv.PagedCache(None, pool[:, 0], pool[:, 1])
    for host, block in (([-1], [0]), ([0], [-1]), (np.array([-1]), [0]), ([0], np.array([-1])), ([0.5], [0]), ([0], [1.0]), ([0], [6]),
                        ([1 << 60], [0]), ([(1 << 64) - 1], [0]), ([[0]], [[0]]), ([True], [0])):
        for f in (c.fetch, c.offload):
            with pytest.raises(ValueError):
                f(1 << 30, host, block)
    half = 16 * 2 * 64 * 2
    for host, block in ((np.array([2], np.int32), [5]), ([2], np.array([5], np.uint64)), (torch.tensor([2]), torch.tensor([5]))):
        e = c._block_entries(1 << 30, host, block, False)
        assert e["src"].tolist() == [(1 << 30) + 4 * half, (1 << 30) + 5 * half]
        assert e["dst"].tolist() == [pool.data_ptr() + 10 * half, pool.data_ptr() + 11 * half]
    assert len(c._block_entries(1 << 30, [], [], False)) == 0


def test_workspace_must_be_contiguous():
    import torch
    pool = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    c = kv.PagedCache(None, pool[:, 0], pool[:, 1])
    i = torch.int32
    b = kv.Batch(torch.zeros(3, dtype=i), torch.zeros(2, dtype=i), torch.zeros(2, 4, dtype=i))
    q, out = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        c.attend(b, q, out, workspace=torch.zeros(64, 1024, dtype=torch.uint8)[:, :512])
