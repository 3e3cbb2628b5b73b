"""Paged KV-cache operators on the GPU against their 64-bit definitions (tests/kv_oracle.py)."""
import ctypes

import numpy as np
import pytest

import gfd_b200
from gfd_b200 import GFD_ERR_INVALID, GfdError, kv
from gfd_b200 import workloads as wl
from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu


def torch_():
    import torch
    return torch


def types():
    torch = torch_()
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class Setup:
    """A random cache, batch and rows.  q_lens / kv_lens: lists.  layout: how the blocks lie."""

    def __init__(self, ctx, dtype, heads, group, d, bt, q_lens, kv_lens, seed, layout="kv_tokens", spare_rows=0, blocks=None,
                 width=None, shared_len=0):
        torch = torch_()
        self.ctx = ctx
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dt = types()[dtype]
        self.d, self.heads, self.hq = d, heads, heads * group
        need = [-(-n // bt) for n in kv_lens]
        shared = -(-shared_len // bt)
        n = blocks or sum(need) + shared + 3
        if layout == "kv_tokens":       # [block][K, V][token][head][d]
            self.pool = self.normal(n, 2, bt, heads, d)
            self.k, self.v = self.pool[:, 0], self.pool[:, 1]
        elif layout == "heads_first":   # [block][head][token][K, V][d]
            self.pool = self.normal(n, heads, bt, 2, d)
            self.k, self.v = (self.pool[:, :, :, i].permute(0, 2, 1, 3) for i in (0, 1))
        elif layout == "apart":         # K and V in tensors of their own, a gap behind every block
            big = [self.normal(n, bt + 1, heads, d) for _ in range(2)]
            self.pool = big
            self.k, self.v = big[0][:, :bt], big[1][:, :bt]
        perm = torch.randperm(n, generator=self.gen, device="cuda").cpu()
        width = width or max(max(need), 1)
        self.table = torch.zeros(len(q_lens), width, dtype=torch.int32)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = perm[at:at + m].int()
            at += m
        self.shared_table = perm[at:at + shared].int().cuda()
        self.table = self.table.cuda()
        self.row_start = [0]
        for m in q_lens:
            self.row_start.append(self.row_start[-1] + m)
        self.q_lens, self.kv_lens = q_lens, kv_lens
        self.rows = self.row_start[-1] + spare_rows
        self.starts = torch.tensor(self.row_start, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        self.cache = kv.PagedCache(ctx, self.k, self.v)
        self.batch = kv.Batch(self.starts, self.lens, self.table)
        self.q = self.normal(self.rows, self.hq, d) * 2
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.shared_len = shared_len

    def normal(self, *shape, dtype=None):
        torch = torch_()
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=dtype or self.dt)

    def workspace(self, max_q_len=0):
        torch = torch_()
        n = self.cache.workspace_bytes(self.rows, self.hq, len(self.q_lens), max_q_len, self.shared_len)
        return torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")  # NaN everywhere

    def attend(self, out_dtype=None, q=None, out=None, want_lse=True, max_q_len=None, stream=None, workspace=None, **kw):
        torch = torch_()
        out = torch.full((self.rows, self.hq, self.d), 7.0, device="cuda", dtype=types()[out_dtype] if out_dtype else self.dt) \
            if out is None else out
        lse = torch.full((self.rows, self.hq), 7.0, device="cuda") if want_lse else None
        mq = max(self.q_lens) if max_q_len is None else max_q_len
        args = dict(lse=lse, max_q_len=mq, workspace=self.workspace(mq) if workspace is None else workspace,
                    status=self.status, stream=stream or torch.cuda.current_stream(), **kw)
        q = self.q if q is None else q
        if self.shared_len:
            self.cache.attend_shared(self.batch, self.shared_table, self.shared_len, q, out, **args)
        else:
            self.cache.attend(self.batch, q, out, **args)
        return out, lse

    def want(self, q=None, scale=None, causal=True, window=0, softcap=0.0, alibi=None, prefix_len=None):
        return oracle.attend(self.k, self.v, self.row_start, self.kv_lens, self.table, self.q if q is None else q,
                             self.d ** -0.5 if scale is None else scale, causal, window, softcap, alibi,
                             None if prefix_len is None else prefix_len.tolist(),
                             self.shared_table if self.shared_len else None, self.shared_len)

    def check(self, out_dtype=None, **kw):
        run = {k: v for k, v in kw.items() if k in ("max_q_len", "want_lse", "workspace", "stream")}
        masks = {k: v for k, v in kw.items() if k not in run}
        out, lse = self.attend(out_dtype=out_dtype, **run, **masks)
        torch_().cuda.synchronize()
        oracle.check_attend(out, lse, self.want(**masks), slice(0, self.row_start[-1]))
        # rows behind the last sequence stay as they were
        assert bool((out[self.row_start[-1]:] == 7).all())
        assert int(self.status) == 0
        return out, lse

    def slopes(self):
        torch = torch_()
        return torch.tensor([2.0 ** (-8.0 * (h + 1) / self.hq) for h in range(self.hq)], device="cuda")

    def ints(self, values):
        return torch_().tensor(values, dtype=torch_().int32, device="cuda")


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def freqs(r):
    torch = torch_()
    return torch.tensor([10000.0 ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float32, device="cuda")


def run_append(s, rot, interleaved, positions=None, with_q=True, stream=None):
    torch = torch_()
    k, v = s.normal(s.rows, s.heads, s.d), s.normal(s.rows, s.heads, s.d)
    before = (s.k.clone(), s.v.clone())
    q_out = torch.full_like(s.q, 7.0) if with_q else None
    s.cache.append(s.batch, k, v, q=s.q if with_q else None, q_out=q_out, inv_freq=freqs(rot) if rot else None,
                   interleaved=interleaved, positions=positions, status=s.status, stream=stream or torch.cuda.current_stream())
    torch.cuda.synchronize()
    return k, v, before, q_out


def check_append(s, rot, interleaved, k, v, before, q_out, positions=None, skip=()):
    """skip: (sequence, row) pairs that must not have been stored."""
    torch = torch_()
    f = freqs(rot) if rot else torch.zeros(0, device="cuda")
    want_k, want_v = before[0].double(), before[1].clone()
    err = torch.zeros_like(want_k)
    bt = s.k.shape[1]
    for i in range(len(s.q_lens)):
        for r in range(s.q_lens[i]):
            if (i, r) in skip:
                continue
            row, pos = s.row_start[i] + r, s.kv_lens[i] - s.q_lens[i] + r
            block, place = int(s.table[i, pos // bt]), pos % bt
            p = torch.tensor([pos if positions is None else int(positions[row])], device="cuda")
            y, e = oracle.rotate(k[row:row + 1], p, f, interleaved)
            want_k[block, place], err[block, place] = y[0], e[0]
            want_v[block, place] = v[row]
            if q_out is not None:
                y, e = oracle.rotate(s.q[row:row + 1], p, f, interleaved)
                oracle.check_rounded(q_out[row:row + 1], y, e)
                if rot < s.d:
                    assert torch.equal(q_out[row, :, rot:], s.q[row, :, rot:])
    assert torch.equal(s.v, want_v)
    still = err == 0
    assert torch.equal(s.k.double()[still], want_k[still])  # copied or untouched: the very bits
    oracle.check_rounded(s.k, want_k, err)
    if q_out is not None:
        assert bool((q_out[s.row_start[-1]:] == 7).all())


@pytest.mark.parametrize("dtype,heads,group,d,bt,rot,interleaved,q_lens,kv_lens,layout", [
    ("bf16", 8, 4, 128, 16, 128, False, [1] * 5, [1, 17, 16, 100, 33], "kv_tokens"),
    ("fp16", 2, 7, 64, 32, 64, True, [3, 0, 40], [3, 5, 200], "heads_first"),
    ("fp16", 1, 1, 128, 48, 32, False, [17, 1], [17, 64], "apart"),
    ("bf16", 3, 2, 64, 16, 16, True, [2, 2, 2], [50, 2, 16], "apart"),
    ("bf16", 1, 5, 64, 16, 0, False, [4], [9], "kv_tokens"),
    ("bf16", 4, 1, 128, 64, 96, True, [700, 600], [1000, 600], "kv_tokens"),
])
def test_append(gpu_ctx, dtype, heads, group, d, bt, rot, interleaved, q_lens, kv_lens, layout):
    s = Setup(gpu_ctx, dtype, heads, group, d, bt, q_lens, kv_lens, seed=len(q_lens) + d, layout=layout, spare_rows=2)
    check_append(s, rot, interleaved, *run_append(s, rot, interleaved))
    assert int(s.status) == 0


def test_append_far_and_given_positions(gpu_ctx):
    """Angles of positions near 2^20 and 2^28 are as accurate as small ones."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 2, 64, 16, [3, 2], [40, 9], seed=5)
    pos = s.ints([0, (1 << 20) - 1, 777777, (1 << 28) + 12345, 5])
    check_append(s, 64, False, *run_append(s, 64, False, positions=pos), positions=pos)


def test_append_q_in_place_and_strided_rows(gpu_ctx):
    torch = torch_()
    s = Setup(gpu_ctx, "fp16", 2, 3, 64, 16, [5, 4], [21, 4], seed=6)
    fused = s.normal(s.rows, s.hq + 2 * s.heads, s.d)  # q, k, v of a row side by side
    q, k, v = fused[:, :s.hq], fused[:, s.hq:s.hq + s.heads], fused[:, s.hq + s.heads:]
    s.q = q.clone()
    before, k0 = (s.k.clone(), s.v.clone()), k.clone()
    s.cache.append(s.batch, k, v, q=q, q_out=q, inv_freq=freqs(64), stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    check_append(s, 64, False, k0, v, before, q)


def test_append_reports_bad_pages_and_lengths(gpu_ctx):
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 1, 64, 16, [2, 2, 2, 2], [18, 18, 18, 18], seed=7)
    s.table[0, 1] = s.cache.blocks       # outside
    s.table[1, 1] = -1                   # outside
    s.lens[2] = 1                        # fewer keys than rows
    s.lens[3] = 33                       # beyond the table
    k, v, before, q_out = run_append(s, 64, False)
    assert int(s.status) == kv.BAD_PAGE | kv.BAD_LENGTH
    assert torch.equal(s.k, before[0]) and torch.equal(s.v, before[1])
    assert bool((q_out[4:] == 7).all()) and not bool((q_out[:4] == 7).any())
    for starts in ([0, 2, 1, 6, 8], [0, 2, 4, 6, 9], [-1, 2, 4, 6, 8]):
        s = Setup(gpu_ctx, "bf16", 2, 1, 64, 16, [2, 2, 2, 2], [18, 18, 18, 18], seed=7)
        s.starts.copy_(s.ints(starts))
        k, v, before, q_out = run_append(s, 64, False)
        assert int(s.status) == kv.BAD_LENGTH
        assert torch.equal(s.k, before[0]) and bool((q_out == 7).all())


# ---------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------
SHAPES = [  # dtype, kv heads, group, d, block tokens, rows of the sequences, keys of the sequences
    ("bf16", 8, 4, 128, 16, [1], [1]),
    ("bf16", 8, 4, 128, 16, [1, 1, 1], [777, 64, 65]),
    ("fp16", 2, 7, 64, 32, [1, 1, 1, 1], [1, 1000, 31, 33]),
    ("bf16", 1, 16, 128, 16, [1] * 9, [5, 300, 16, 17, 15, 128, 127, 129, 2]),
    ("fp16", 3, 3, 128, 48, [2, 0, 5, 1], [100, 7, 5, 259]),
    ("bf16", 2, 1, 64, 64, [16, 3], [500, 90]),
    ("bf16", 2, 4, 128, 16, [130, 1, 70], [130, 200, 333]),
    ("fp16", 1, 8, 64, 16, [64], [64]),
    ("bf16", 1, 2, 128, 1024, [300], [1300]),
    ("fp16", 2, 5, 64, 16, [257, 40], [600, 41]),
    ("bf16", 1, 40, 64, 16, [1, 7], [50, 70]),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attend(gpu_ctx, shape):
    s = Setup(gpu_ctx, *SHAPES[shape], seed=shape, spare_rows=2)
    s.check()


MASKS = [
    dict(window=1), dict(window=20), dict(causal=False), dict(causal=False, window=33), dict(softcap=5.0),
    dict(alibi=True), dict(prefix=[3]), dict(prefix=[40], window=17), dict(prefix=[100000], softcap=20.0),
    dict(prefix=[-5], window=64, alibi=True, softcap=30.0), dict(scale=0.3), dict(scale=0.0), dict(scale=-0.1),
]


@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("shape", [1, 2, 4, 6, 9])
def test_attend_masks(gpu_ctx, shape, mask):
    s = Setup(gpu_ctx, *SHAPES[shape], seed=100 + shape)
    kw = dict(MASKS[mask])
    if kw.pop("alibi", False):
        kw["alibi"] = s.slopes()
    if "prefix" in kw:
        kw["prefix_len"] = s.ints((kw.pop("prefix") * len(s.q_lens))[:len(s.q_lens)])
    s.check(**kw)


@pytest.mark.parametrize("layout", ["heads_first", "apart"])
@pytest.mark.parametrize("shape", [1, 4, 6])
def test_attend_layouts_and_types(gpu_ctx, shape, layout):
    s = Setup(gpu_ctx, *SHAPES[shape], seed=200 + shape, layout=layout)
    s.check(out_dtype="fp32")
    s.check(want_lse=False)
    s.check(max_q_len=0)


@pytest.mark.parametrize("shape", [2, 6])
def test_attend_strided_rows(gpu_ctx, shape):
    torch = torch_()
    s = Setup(gpu_ctx, *SHAPES[shape], seed=300 + shape)
    wide = s.normal(s.hq + 3, s.rows, s.d + 8)  # heads outermost, gaps
    q = wide[1:1 + s.hq, :, :s.d].permute(1, 0, 2)
    room = torch.full((s.rows, 2 * s.hq, s.d), 7.0, device="cuda", dtype=s.dt)
    out = room[:, ::2]
    got, lse = s.attend(q=q, out=out)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, s.want(q=q))
    assert bool((room[:, 1::2] == 7).all())
    one = s.normal(s.rows, 1, s.d).expand(s.rows, s.hq, s.d)  # one head broadcast to all
    got, lse = s.attend(q=one)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, s.want(q=one))


@pytest.mark.parametrize("shape", [1, 3, 4, 6, 9])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_attend_ignores_what_is_masked(gpu_ctx, shape, poison):
    """NaN and infinities in every place no row sees, and in places that only some rows see."""
    torch = torch_()
    s = Setup(gpu_ctx, *SHAPES[shape], seed=400 + shape)
    clean = (s.k.clone(), s.v.clone())
    want = s.want(window=30)
    bt = s.k.shape[1]
    mine = torch.zeros(s.cache.blocks, bt, dtype=torch.bool, device="cuda")
    for i, n in enumerate(s.kv_lens):
        for j in range(max(0, n - s.q_lens[i] - 29), n):
            mine[int(s.table[i, j // bt]), j % bt] = True
    s.k[~mine], s.v[~mine] = poison, poison
    got, lse = s.attend(window=30)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, want)
    # the last key of the longest sequence is seen by its last row alone
    s.k.copy_(clean[0]), s.v.copy_(clean[1])
    i = max(range(len(s.q_lens)), key=lambda x: s.q_lens[x])
    j = s.kv_lens[i] - 1
    s.v[int(s.table[i, j // bt]), j % bt] = poison
    got, lse = s.attend(window=30)
    torch.cuda.synchronize()
    last = s.row_start[i + 1] - 1
    rows = [r for r in range(s.row_start[-1]) if r != last]
    oracle.check_attend(got, lse, want, rows)
    assert not bool(torch.isfinite(got[last].float()).any())


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [3000, 500]), ([2000, 40], [2100, 300])])
def test_attend_nan_that_is_seen(gpu_ctx, q_lens, kv_lens):
    """A NaN or an infinity that rows see makes those rows NaN or infinite and no others, and does
    not cost more than a few times the call."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, q_lens, kv_lens, seed=17)
    want = s.want(window=700)
    n = s.row_start[-1]
    s.q[q_lens[0] // 2] = float("nan")
    got, lse = s.attend(window=700)
    torch.cuda.synchronize()
    assert bool(torch.isnan(got[q_lens[0] // 2].float()).all()) and bool(torch.isnan(lse[q_lens[0] // 2]).all())
    oracle.check_attend(got, lse, want, [r for r in range(n) if r != q_lens[0] // 2])
    s.q[:] = torch.where(torch.isnan(s.q), torch.zeros_like(s.q), s.q)
    want = s.want(window=700)
    j = kv_lens[0] - q_lens[0] // 2 - 650  # seen by some rows only
    s.v[int(s.table[0, j // 16]), j % 16, :, 5] = float("nan")
    got, lse = s.attend(window=700)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    sees = [r for r in range(q_lens[0]) if j <= kv_lens[0] - q_lens[0] + r < j + 700]
    assert sees and bool(torch.isnan(got[sees][:, :, 5].float()).all())
    oracle.check_attend(got[:, :, 6:], lse, tuple(x[:, :, 6:] if x.dim() == 3 else x for x in want))
    oracle.check_attend(got, lse, want, [r for r in range(n) if r not in set(sees)])


@pytest.mark.parametrize("q_lens,kv_lens", [([3], [500]), ([400], [700])])
def test_attend_nan_seen_in_one_element_and_masked_in_another(gpu_ctx, q_lens, kv_lens):
    torch = torch_()
    s = Setup(gpu_ctx, "fp16", 2, 4, 128, 16, q_lens, kv_lens, seed=23)
    want = s.want()
    s.v[int(s.table[0, 1]), 3, :, 5] = float("nan")  # every row sees it
    j = kv_lens[0] - 1  # the last row alone sees it
    s.v[int(s.table[0, j // 16]), j % 16, :, 77] = float("inf")
    got, lse = s.attend()
    torch.cuda.synchronize()
    assert bool(torch.isnan(got[:, :, 5].float()).all()) and bool(torch.isinf(got[-1, :, 77].float()).all())
    n = q_lens[0]
    keep = [d for d in range(128) if d not in (5, 77)]
    cut = lambda x, d: x[:, :, d] if x.dim() == 3 else x
    oracle.check_attend(got[:, :, keep], lse, tuple(cut(x, keep) for x in want))
    oracle.check_attend(got[:, :, 77:78], lse, tuple(cut(x, [77]) for x in want), list(range(n - 1)))


def test_attend_all_values_nan_is_not_slow(gpu_ctx):
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, [4000], [4000], seed=18)
    s.v[:] = float("nan")
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    s.attend()
    a.record()
    got, _ = s.attend()
    b.record()
    torch.cuda.synchronize()
    assert bool(torch.isnan(got.float()).all()) and int(s.status) == 0
    assert a.elapsed_time(b) < 100  # the call itself takes 0.3 ms


@pytest.mark.parametrize("shape", [1, 4, 6])
def test_attend_pages_behind_the_window_may_be_gone(gpu_ctx, shape):
    """Block ids of pages that no row sees are not looked at."""
    torch = torch_()
    s = Setup(gpu_ctx, *SHAPES[shape], seed=19)
    bt = s.k.shape[1]
    want = s.want(window=20)
    for i, n in enumerate(s.kv_lens):
        first = max(0, n - s.q_lens[i] - 19) // bt
        s.table[i, :first] = -1
        s.table[i, -(-n // bt):] = 2 ** 31 - 1
    got, lse = s.attend(window=20)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    oracle.check_attend(got, lse, want)


def test_attend_bad_pages_are_masked(gpu_ctx):
    torch = torch_()
    for shape in (1, 6):
        s = Setup(gpu_ctx, *SHAPES[shape], seed=500)
        s.table[0, 1] = s.cache.blocks
        s.table[0, 3] = -7
        s.table[1, :] = 2 ** 31 - 1  # a sequence whose pages are all bad: nothing to see
        got, lse = s.attend()
        torch.cuda.synchronize()
        assert int(s.status) == kv.BAD_PAGE
        oracle.check_attend(got, lse, s.want())
        a, b = s.row_start[1], s.row_start[2]
        assert bool((got[a:b] == 0).all()) and bool((lse[a:b] == float("-inf")).all())


def test_attend_bad_lengths_skip_the_sequence(gpu_ctx):
    torch = torch_()
    for shape in (1, 6):
        s = Setup(gpu_ctx, *SHAPES[shape], seed=501)
        want = s.want()
        s.lens[1] = 100000
        got, lse = s.attend()
        torch.cuda.synchronize()
        a, b = s.row_start[1], s.row_start[2]
        assert int(s.status) == kv.BAD_LENGTH and bool((got[a:b] == 7).all()) and bool((lse[a:b] == 7).all())
        oracle.check_attend(got, lse, want, [r for r in range(s.rows) if not a <= r < b])
        s.lens[1] = -1
        got, _ = s.attend()
        assert bool((got[a:b] == 7).all())
        s.starts[1] = s.rows + 1
        got, _ = s.attend()
        assert bool((got == 7).all())
    s = Setup(gpu_ctx, *SHAPES[6], seed=502)
    got, _ = s.attend(max_q_len=100)  # the first sequence has 130 rows
    assert int(s.status) == kv.BAD_LENGTH and bool((got[:130] == 7).all())
    oracle.check_attend(got, None, s.want(), slice(130, None))


def test_attend_same_block_twice(gpu_ctx):
    """A table may name a block more than once, and sequences may share blocks."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, [1, 3], [100, 90], seed=8)
    s.table[1, :4] = s.table[0, :4]
    s.table[0, 2] = s.table[0, 1]
    s.check()


def test_attend_offsets_past_32_bits(gpu_ctx):
    """Blocks whose elements lie beyond 2^32 bytes and beyond 2^31 elements of the cache."""
    torch = torch_()
    n, bt, h, d = 70000, 16, 8, 128
    pool = torch.empty(n, 2, bt, h, d, dtype=torch.bfloat16, device="cuda")  # 4.6 GB
    s = Setup(gpu_ctx, "bf16", h, 2, d, bt, [1, 40], [100, 150], seed=9)
    high = n - 1 - torch.arange(s.cache.blocks, device="cuda")
    pool[high] = s.pool
    s.table = (n - 1 - s.table).int()
    s.k, s.v = pool[:, 0], pool[:, 1]
    s.cache = kv.PagedCache(gpu_ctx, s.k, s.v)
    s.batch = kv.Batch(s.starts, s.lens, s.table)
    s.check()
    del pool


def test_attend_many_sequences(gpu_ctx):
    """More sequences than threads of a block, most of them short, some without rows."""
    rng = np.random.default_rng(3)
    q = [int(x) for x in rng.integers(0, 3, 700)]
    s = Setup(gpu_ctx, "fp16", 1, 2, 64, 16, q, [n + int(x) for n, x in zip(q, rng.integers(0, 40, 700))], seed=10)
    s.check()


def test_attend_long(gpu_ctx):
    s = Setup(gpu_ctx, "bf16", 1, 4, 128, 16, [1, 2], [20001, 9000], seed=11)
    s.check()
    s.check(alibi=s.slopes(), softcap=50.0)


# ---------------------------------------------------------------------------
# attend_shared
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,heads,group,d,bt,q_lens,kv_lens,shared,kw", [
    ("bf16", 8, 4, 128, 16, [1] * 9, [1, 50, 16, 17, 3, 2, 64, 65, 90], 1000, {}),
    ("fp16", 4, 5, 64, 16, [3] * 7, [3, 9, 16, 17, 60, 33, 4], 111, {}),
    ("bf16", 1, 8, 64, 32, [1, 0, 40, 2], [1, 3, 90, 7], 5, {}),
    ("bf16", 2, 3, 128, 16, [1, 2, 3], [30, 31, 32], 257, dict(window=100)),
    ("fp16", 2, 3, 64, 48, [1, 2, 150], [30, 31, 170], 300, dict(softcap=10.0, alibi=True)),
    ("bf16", 2, 1, 128, 16, [5, 2], [5, 2], 64, dict(causal=False)),
    ("bf16", 2, 1, 128, 16, [5, 2], [50, 20], 64, dict(window=30, prefix=[7, 70])),
])
def test_attend_shared(gpu_ctx, dtype, heads, group, d, bt, q_lens, kv_lens, shared, kw):
    s = Setup(gpu_ctx, dtype, heads, group, d, bt, q_lens, kv_lens, seed=shared, spare_rows=1, shared_len=shared)
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi"] = s.slopes()
    if "prefix" in kw:
        kw["prefix_len"] = s.ints(kw.pop("prefix"))
    s.check(**kw)
    s.check(out_dtype="fp32", **kw)


def test_shared_equals_tables_that_name_it(gpu_ctx):
    """The same context written as one table per sequence gives the same result within bounds."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, [1, 2, 1], [33, 20, 1], seed=12, shared_len=160)
    a, la = s.attend()
    n = 160 // 16
    t = torch.cat([s.shared_table[None].expand(3, n), s.table], 1).contiguous()
    whole = kv.Batch(s.starts, (s.lens + 160).int(), t)
    b, lb = torch.empty_like(a), torch.empty_like(la)
    ws = torch.empty(max(16, s.cache.workspace_bytes(s.rows, s.hq, 3, 2)), dtype=torch.uint8, device="cuda")
    s.cache.attend(whole, s.q, b, lse=lb, max_q_len=2, workspace=ws, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = s.want()
    oracle.check_attend(a, la, want)
    oracle.check_attend(b, lb, want)


def test_shared_masks_poison_and_bad_pages(gpu_ctx):
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, [1, 2, 60], [9, 20, 70], seed=13, shared_len=100)
    used = int(s.shared_table[-1])
    s.k[used, 100 % 16:], s.v[used, 100 % 16:] = float("nan"), float("inf")
    s.check()
    s.shared_table[2] = -1
    got, lse = s.attend()
    torch.cuda.synchronize()
    assert int(s.status) == kv.BAD_PAGE
    oracle.check_attend(got, lse, s.want())


@pytest.mark.parametrize("q_lens", [[1, 2, 1], [1, 2, 60], [300, 2, 60]])
def test_shared_bad_lengths_skip_the_sequence(gpu_ctx, q_lens):
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, q_lens, [n + 9 for n in q_lens], seed=16, spare_rows=1, shared_len=700)
    want = s.want()
    s.lens[1] = 1  # fewer keys than rows
    got, lse = s.attend()
    torch.cuda.synchronize()
    a, b = s.row_start[1], s.row_start[2]
    assert int(s.status) == kv.BAD_LENGTH and bool((got[a:b] == 7).all()) and bool((lse[a:b] == 7).all())
    oracle.check_attend(got, lse, want, [r for r in range(s.row_start[-1]) if not a <= r < b])
    s.starts[1] = s.rows + 5
    got, lse = s.attend()
    torch.cuda.synchronize()
    assert bool((got == 7).all()) and bool((lse == 7).all())


# ---------------------------------------------------------------------------
# merge
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("part,out,n,rows,heads,d", [
    ("bf16", "bf16", 2, 5, 4, 128), ("fp32", "bf16", 3, 1, 1, 64), ("fp16", "fp32", 8, 33, 7, 64),
    ("fp32", "fp32", 1, 17, 5, 128), ("fp32", "fp16", 37, 3, 2, 128),
])
def test_merge(gpu_ctx, part, out, n, rows, heads, d):
    torch = torch_()
    gen = torch.Generator(device="cuda").manual_seed(n)
    parts = torch.randn(n, rows, heads, d, generator=gen, device="cuda").to(types()[part])
    lse = torch.randn(n, rows, heads, generator=gen, device="cuda") * 10
    if n > 1:
        lse[0, 0] = float("-inf")       # a part that saw nothing: its output is not read
        parts[0, 0] = float("nan")
        lse[:, rows - 1, heads - 1] = float("-inf")
    o = torch.full((rows, heads, d), 7.0, device="cuda", dtype=types()[out])
    l = torch.full((rows, heads), 7.0, device="cuda")
    kv.merge(gpu_ctx, parts, lse, o, lse=l, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    want, wl_, tol, ltol = oracle.merge(parts, lse, types()[out])
    oracle.check_rounded(o, want, tol)
    none = torch.isinf(wl_)
    assert torch.equal(l.double()[none], wl_[none]) and bool((o[none] == 0).all())
    assert bool(((l.double() - wl_)[~none].abs() <= ltol[~none]).all())


def test_merge_strides_and_no_rows(gpu_ctx):
    torch = torch_()
    gen = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(4, 6, 3, 2, 64, generator=gen, device="cuda").to(torch.bfloat16)
    parts = big[:, :, :, 1].permute(0, 2, 1, 3)  # [4, 3, 6, 64], strided
    lse = torch.randn(4, 3, 6, generator=gen, device="cuda")
    o = torch.empty(6, 3, 64, device="cuda", dtype=torch.bfloat16).permute(1, 0, 2)
    kv.merge(gpu_ctx, parts, lse, o, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    want, _, tol, _ = oracle.merge(parts, lse, torch.bfloat16)
    oracle.check_rounded(o, want, tol)
    kv.merge(gpu_ctx, parts[:, :0], lse[:, :0].contiguous(), o[:0], stream=torch.cuda.current_stream())


# ---------------------------------------------------------------------------
# Together, on streams, in graphs
# ---------------------------------------------------------------------------
def test_fetch_append_attend_merge(gpu_ctx):
    """A decode step over blocks that come from host memory: half of each context is fetched,
    attended apart and merged with the resident half; the step's own rows are appended first."""
    torch = torch_()
    stream = torch.cuda.Stream()
    bt, h, d, g = 16, 8, 128, 4
    nblk = 64
    blk = 2 * bt * h * d
    host = gpu_ctx.pool(nblk * blk * 2)
    wl.fill_bf16_normal(host.ptr, nblk * blk, 7)
    src = torch.from_numpy(host.array(np.int16).copy()).view(torch.bfloat16).view(nblk, 2, bt, h, d).cuda()
    kvs = [97, 160, 33]
    s = Setup(gpu_ctx, "bf16", h, g, d, bt, [1, 1, 1], kvs, seed=14, blocks=40)
    # the first blocks of every sequence come from the host pool
    near = [n // 2 // bt for n in kvs]
    ids, hosts = [], []
    for i, n in enumerate(near):
        ids += s.table[i, :n].tolist()
        hosts += [(7 * (len(hosts) + x)) % nblk for x in range(n)]
    torch.cuda.synchronize()
    s.cache.fetch(host.ptr, hosts, ids, stream=stream)
    k, v = s.normal(3, h, d), s.normal(3, h, d)
    q_rot = torch.empty_like(s.q)
    torch.cuda.synchronize()
    s.cache.append(s.batch, k, v, q=s.q, q_out=q_rot, inv_freq=freqs(d), stream=stream)
    far = kv.Batch(s.starts, s.ints([n * bt for n in near]), s.table)                       # the fetched part
    rest = torch.stack([torch.roll(s.table[i], -near[i]) for i in range(3)]).contiguous()
    here = kv.Batch(s.starts, s.ints([n - m * bt for n, m in zip(kvs, near)]), rest)        # the resident part
    parts = torch.empty(2, 3, s.hq, d, device="cuda")
    lses = torch.empty(2, 3, s.hq, device="cuda")
    out, lse = torch.empty_like(s.q), torch.empty(3, s.hq, device="cuda")
    ws = s.workspace(1)
    torch.cuda.synchronize()
    s.cache.attend(far, q_rot, parts[0], lse=lses[0], causal=False, max_q_len=1, workspace=ws, stream=stream)
    s.cache.attend(here, q_rot, parts[1], lse=lses[1], max_q_len=1, workspace=ws, stream=stream)
    kv.merge(gpu_ctx, parts, lses, out, lse=lse, stream=stream)
    stream.synchronize()
    for a, b in zip(ids, hosts):
        assert torch.equal(s.pool[a], src[b])
    want = s.want(q=q_rot)
    # the parts' own bounds carry over with their weights; the merge adds its roundings
    o, l, tol, ltol = want
    slack = 2.0 ** -18 * (1 + 2 * l.abs()).amax()
    oracle.check_attend(out, lse, (o, l, tol * 2 + o.abs().amax() * slack, ltol * 2 + slack))
    s.cache.offload(host.ptr, hosts[:1], ids[:1], stream=stream)
    stream.synchronize()
    host.free()


@pytest.mark.parametrize("shape", [1, 6])
def test_graph_reads_lengths_at_replay(gpu_ctx, shape):
    """A captured step replayed with other lengths, tables and rows; two graphs with a workspace
    each, replayed side by side."""
    torch = torch_()
    a, b = (Setup(gpu_ctx, *SHAPES[shape], seed=600 + i) for i in (0, 1))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for s, st in zip((a, b), streams):
        ws = s.workspace(max(s.q_lens))
        out = torch.empty_like(s.q)
        lse = torch.empty(s.rows, s.hq, device="cuda")
        kw = dict(lse=lse, max_q_len=max(s.q_lens), workspace=ws, stream=st)
        torch.cuda.synchronize()
        s.cache.attend(s.batch, s.q, out, **kw)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.cache.attend(s.batch, s.q, out, **kw)
        runs.append((g, out, lse, ws))  # a graph holds addresses: its workspace lives as long
    for s in (a, b):  # other inputs in the same arrays
        s.q.copy_(s.normal(*s.q.shape))
        s.kv_lens = [n - 3 if n > 60 and m < n - 3 else n for n, m in zip(s.kv_lens, s.q_lens)]
        s.lens.copy_(s.ints(s.kv_lens))
        s.table.copy_(torch.flip(s.table, [0]) if len(set(-(-n // s.k.shape[1]) for n in s.kv_lens)) == 1 else s.table)
    torch.cuda.synchronize()
    for _ in range(3):
        for (g, _, _, _), st in zip(runs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, (g, out, lse, _) in zip((a, b), runs):
        oracle.check_attend(out, lse, s.want())


@pytest.mark.parametrize("shape", [3, 9])
def test_same_inputs_same_bits(gpu_ctx, shape):
    torch = torch_()
    s = Setup(gpu_ctx, *SHAPES[shape], seed=700)
    ref, rl = s.attend()
    for _ in range(5):
        out, lse = s.attend()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(lse, rl)


def test_context_stream_and_threads(gpu_ctx):
    """stream 0 is the context's stream; calls from several threads are serialised."""
    import threading
    torch = torch_()
    sets = [Setup(gpu_ctx, *SHAPES[i], seed=800 + i) for i in (1, 4, 6)]
    outs = [torch.empty_like(s.q) for s in sets]
    works = [s.workspace(0) for s in sets]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=lambda s=s, o=o, w=w: [s.cache.attend(s.batch, s.q, o, workspace=w) for _ in range(20)])
               for s, o, w in zip(sets, outs, works)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s, o in zip(sets, outs):
        oracle.check_attend(o, None, s.want())


# ---------------------------------------------------------------------------
# Refusals that need device pointers
# ---------------------------------------------------------------------------
def test_refusals(gpu_ctx):
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 2, 64, 16, [1, 1], [20, 30], seed=15)
    out = torch.full_like(s.q, 7.0)
    ws = s.workspace(1)

    def refused(f, *a, **kw):
        with pytest.raises(GfdError) as e:
            f(*a, **kw)
        assert e.value.code == GFD_ERR_INVALID
        return str(e.value)

    def attend(q=s.q, o=out, batch=s.batch, **kw):
        s.cache.attend(batch, q, o, **{**dict(max_q_len=1, workspace=ws), **kw})

    assert "out must not be q" in refused(attend, o=s.q)
    assert "not inside one device allocation" in refused(attend, q=s.q.cpu())
    assert "not inside one device allocation" in refused(attend, o=out.cpu())
    assert "not inside one device allocation" in refused(attend, lse=torch.zeros(2, 4))
    host = kv.Batch(s.starts.cpu(), s.lens, s.table)
    assert "row_start" in refused(attend, batch=host)
    assert "table" in refused(attend, batch=kv.Batch(s.starts, s.lens, s.table.cpu()))
    odd = torch.empty(2 * 4 * 64 + 8, device="cuda", dtype=torch.bfloat16)[1:1 + 512].view(2, 4, 64)
    assert "aligned" in refused(attend, q=odd)
    gap = torch.empty(2, 4, 68, device="cuda", dtype=torch.bfloat16)[:, :, :64]
    assert "multiples of 8" in refused(attend, q=gap)
    assert "overlap" in refused(attend, o=torch.empty(1, 4, 64, device="cuda", dtype=torch.bfloat16).expand(2, 4, 64))
    for kw in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(scale=float("nan")), dict(window=-1), dict(max_q_len=-1)):
        refused(attend, **kw)
    k, v = s.normal(2, 2, 64), s.normal(2, 2, 64)
    assert "not inside one device allocation" in refused(s.cache.append, s.batch, k.cpu(), v)
    assert "rot_dim" in refused(s.cache.append, s.batch, k, v, inv_freq=torch.zeros(5, device="cuda"))
    both = kv.PagedCache(gpu_ctx, s.k, s.k)
    assert "same array" in refused(both.append, s.batch, k, v)
    parts = torch.zeros(2, 1, 1, 64, device="cuda")
    assert "out must not be a part" in refused(kv.merge, gpu_ctx, parts, torch.zeros(2, 1, 1, device="cuda"), parts[1])
    torch.cuda.synchronize()
    assert bool((out == 7).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,group", [(3, 1), (2, 3), (1, 7), (2, 16), (1, 128), (1, 160)])
def test_attend_prompt_groups(gpu_ctx, heads, group, d):
    """Units of 128 packed rows of a half begin inside a token's heads or not, with the next
    sequence's rows behind the last one: NaN there reaches nothing."""
    rows = [max(2, 300 // group), 1, max(3, 520 // group + 1)]
    s = Setup(gpu_ctx, "bf16", heads, group, d, 16, rows, [n + 45 for n in rows], seed=29)
    s.check()
    s.q[rows[0]:] = float("nan")
    got, lse = s.attend()
    torch_().cuda.synchronize()
    assert bool(torch_().isnan(got[rows[0]:].float()).all())
    s.q[rows[0]:] = 0
    oracle.check_attend(got, lse, s.want(), slice(0, rows[0]))


@pytest.mark.parametrize("kind", ["heads_first", "broadcast_rows", "broadcast_heads", "gap"])
def test_attend_prompt_q_strides(gpu_ctx, kind):
    torch = torch_()
    s = Setup(gpu_ctx, "fp16", 2, 4, 128, 16, [200, 70], [300, 70], seed=31)
    n, h = s.q.shape[:2]
    if kind == "heads_first":
        q = s.normal(h, n, 128).transpose(0, 1)
    elif kind == "broadcast_rows":
        q = s.normal(1, h, 128).expand(n, h, 128)
    elif kind == "broadcast_heads":
        q = s.normal(n, 1, 128).expand(n, h, 128)
    else:
        q = s.normal(n, h + 1, 136)[:, 1:, 8:]
    got, lse = s.attend(q=q)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, s.want(q=q))


@pytest.mark.parametrize("out_dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_prompt_rows_off_32_bytes(gpu_ctx, d, out_dtype):
    """Result rows that begin on 16 bytes and not on 32."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, d, 32, [150, 20], [150, 333], seed=37)
    e = 4 if out_dtype == "fp32" else 8
    big = torch.full((s.rows, s.hq, d + 2 * e), 7.0, device="cuda", dtype=types()[out_dtype])
    out = big[:, :, e:e + d]
    assert out.data_ptr() % 32 == 16
    got, lse = s.attend(out=out)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, s.want())
    assert bool((big[:, :, :e] == 7).all()) and bool((big[:, :, e + d:] == 7).all())


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 4], [700, 40]), ([130, 60], [400, 60])])
def test_attend_cap_of_large_scores(gpu_ctx, q_lens, kv_lens):
    """Scores far above the cap next to ones below it."""
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, q_lens, kv_lens, seed=41)
    s.q[:, ::2] *= 6
    s.check(softcap=2.0)
    s.check(softcap=500.0, scale=-0.25)


def test_attend_padded_batch(gpu_ctx):
    """Empty sequences before, between and behind, whatever their lengths and tables say, and rows of none."""
    torch = torch_()
    q_lens, kv_lens = [0, 90, 0, 0, 1, 0, 3, 0], [0, 90, 0, 0, 50, 0, 64, 0]
    s = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, q_lens, kv_lens, seed=43, spare_rows=9)
    empty = [i for i, n in enumerate(q_lens) if n == 0]
    s.lens[empty] = torch.tensor([0, -5, 10 ** 9, 7, 1], dtype=torch.int32, device="cuda")
    s.table[empty] = -1
    s.check()
    none = kv.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), s.lens[:0], s.table[:0])
    out = torch.full_like(s.q, 7.0)
    s.cache.attend(none, s.q, out, workspace=s.workspace(), status=s.status)
    s.cache.attend(s.batch, s.q[:0], out[:0], workspace=s.workspace(), status=s.status)
    torch.cuda.synchronize()
    assert bool((out == 7).all()) and int(s.status) in (0, kv.BAD_LENGTH)


def test_attend_4096_sequences(gpu_ctx):
    rng = np.random.default_rng(47)
    q_lens = [int(x) for x in rng.integers(0, 3, 4096)]
    q_lens[1000], q_lens[4095] = 70, 33
    s = Setup(gpu_ctx, "fp16", 1, 2, 64, 16, q_lens, [n + int(x) for n, x in zip(q_lens, rng.integers(0, 30, 4096))], seed=47)
    s.check()


def test_shared_on_two_streams_and_in_a_graph(gpu_ctx):
    """Two calls at once, each with its workspace, and one replayed behind a changed prefix."""
    torch = torch_()
    a = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, [1, 5, 1], [9, 70, 33], seed=53, shared_len=500)
    b = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, [40, 2], [60, 2], seed=54, shared_len=260)
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    res = []
    for _ in range(20):
        res = []
        for s, x in zip((a, b), st):
            with torch.cuda.stream(x):  # the results and workspaces are filled there too
                res.append(s.attend())
    torch.cuda.synchronize()
    for s, (out, lse) in zip((a, b), res):
        oracle.check_attend(out, lse, s.want())
    out, lse, ws = torch.empty_like(a.q), torch.empty(a.rows, a.hq, device="cuda"), a.workspace(5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.cache.attend_shared(a.batch, a.shared_table, a.shared_len, a.q, out, lse=lse, max_q_len=5, workspace=ws, status=a.status,
                              stream=torch.cuda.current_stream())
    a.q.normal_(generator=a.gen)
    a.shared_table[:] = a.shared_table.flip(0)
    a.lens[1] = a.kv_lens[1] = 12
    g.replay()
    torch.cuda.synchronize()
    oracle.check_attend(out, lse, a.want())
    assert int(a.status) == 0


def put(s, i, j, e, value):
    """V of key j of sequence i, element(s) e of every head."""
    bt = s.k.shape[1]
    s.v[int(s.table[i, j // bt]), j % bt, :, e] = value


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("seen", [INF, -INF])
@pytest.mark.parametrize("masked", [NAN, INF, -INF])
@pytest.mark.parametrize("dtype,d,q_lens,kv_lens", [("bf16", 64, [4], [45]), ("fp16", 128, [3], [500]), ("fp16", 64, [150], [200]),
                                                    ("bf16", 128, [70], [1000])])
def test_attend_seen_infinity_beside_a_masked_value(gpu_ctx, dtype, d, q_lens, kv_lens, seen, masked):
    """An infinity that a row sees is its result in that element, whatever the same element of a masked key holds."""
    torch = torch_()
    s = Setup(gpu_ctx, dtype, 2, 4, d, 16, q_lens, kv_lens, seed=61)
    want = s.want()
    n, keys = q_lens[0], kv_lens[0]
    put(s, 0, keys - n, 9, seen)          # every row sees it
    put(s, 0, keys - 1, 9, masked)        # the last row alone sees this one
    put(s, 0, keys - n // 2, 33, -seen)   # the rows of the first half do not see this one
    put(s, 0, keys - 1, 33, masked)
    put(s, 0, keys - n, d - 1, seen)      # NaN by what every row sees
    put(s, 0, keys - n, d - 2, NAN)
    put(s, 0, max(0, keys - n - 1), d - 1, -seen)
    put(s, 0, keys - 1, d - 1, masked)
    got, lse = s.attend()
    torch.cuda.synchronize()
    assert int(s.status) == 0
    rows = list(range(n - 1))             # all but the last
    g = got.float()
    assert bool((g[rows, :, 9] == seen).all())
    last = seen if masked == seen else NAN
    assert bool((g[n - 1, :, 9] == last).all() if last == seen else torch.isnan(g[n - 1, :, 9]).all())
    half = [r for r in rows if r >= n - n // 2]  # row i stands at keys - n + i
    assert bool((g[half, :, 33] == -seen).all())
    assert bool(torch.isnan(g[:, :, d - 2:]).all())
    keep = [e for e in range(d) if e not in (9, 33, d - 1, d - 2)]
    oracle.check_attend(got[:, :, keep], lse, tuple(x[:, :, keep] if x.dim() == 3 else x for x in want))
    before = [r for r in rows if r < n - n // 2]
    oracle.check_attend(got[:, :, 33:34], lse, tuple(x[:, :, 33:34] if x.dim() == 3 else x for x in want), before)


@pytest.mark.parametrize("masked", [NAN, INF, -INF])
@pytest.mark.parametrize("d,q_lens", [(64, [2, 5, 1]), (128, [2, 130, 3])])
def test_shared_seen_infinity_beside_a_masked_value(gpu_ctx, d, q_lens, masked):
    """The same in a shared prefix: a window hides its first keys from some rows only."""
    torch = torch_()
    kv_lens = [n + 7 for n in q_lens]
    s = Setup(gpu_ctx, "bf16", 2, 4, d, 16, q_lens, kv_lens, seed=62, shared_len=200)
    window = 60  # both values in the same keys of a tile
    want = s.want(window=window)
    first = [200 + n - m + i - window + 1 for n, m in zip(kv_lens, q_lens) for i in range(m)]  # first key each row sees
    at = int(s.shared_table[199 // 16])
    s.v[at, 199 % 16, :, 9] = INF                         # seen by all rows whose window reaches back so far
    j = min(first)                                        # seen by the row that sees furthest back
    s.v[int(s.shared_table[j // 16]), j % 16, :, 9] = masked
    got, lse = s.attend(window=window)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    g = got.float()
    sees = [r for r, f in enumerate(first) if j < f <= 199]
    none = [r for r, f in enumerate(first) if f > 199]
    assert sees and bool((g[sees, :, 9] == INF).all())
    keep = [e for e in range(d) if e != 9]
    oracle.check_attend(got[:, :, keep], lse, tuple(x[:, :, keep] if x.dim() == 3 else x for x in want))
    if none:
        oracle.check_attend(got, lse, want, none)


@pytest.mark.parametrize("out_dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,q_lens,kv_lens", [(64, [4, 3], [60, 900]), (128, [3, 4], [2000, 21]), (64, [90, 2], [300, 33]),
                                              (128, [130], [3000])])
def test_attend_rows_summed_again_replace_the_first_sums(gpu_ctx, d, q_lens, kv_lens, out_dtype):
    """Rows that a masked NaN reached are written twice; the second time is what stays, call after call."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 4, d, 16, q_lens, kv_lens, seed=63)
    want = s.want()
    ends = [b - 1 for b in s.row_start[1:]]
    for i, n in enumerate(kv_lens):
        put(s, i, n - 1, slice(None), NAN)  # the last row of each sequence alone sees it
    rows = [r for r in range(s.rows) if r not in ends]
    first = None
    for _ in range(30):
        got, lse = s.attend(out_dtype=out_dtype)
        torch.cuda.synchronize()
        first = got.clone() if first is None else first
        assert torch.equal(got[rows], first[rows])
    oracle.check_attend(got, lse, want, rows)
    assert bool(torch.isnan(got[ends].float()).all())


@pytest.mark.parametrize("field,value", [("heads", 0), ("heads", -3), ("heads", 1025), ("head_dim", 0), ("block_tokens", 0), ("blocks", 0),
                                         ("dtype", 7)])
def test_entry_points_refuse_a_cache_of_no_shape(gpu_ctx, field, value):
    """Through the C entry points: nothing is worked out from a shape before it is checked."""
    s = Setup(gpu_ctx, "bf16", 2, 2, 64, 16, [1, 1], [20, 30], seed=64)
    c = kv._Cache.from_buffer_copy(s.cache._c)
    setattr(c, field, value)
    l, h, b = gpu_ctx.lib, gpu_ctx.handle, s.batch._c(2)
    out, ws = torch_().full_like(s.q, 7.0), s.workspace(1)
    a = kv._Attend(q=kv._Rows(s.q.data_ptr(), 256, 64), out=kv._Rows(out.data_ptr(), 256, 64), workspace=ws.data_ptr(),
                   workspace_bytes=ws.numel(), q_heads=4, scale=0.1, out_dtype=kv.BF16)
    n = ctypes.c_size_t()
    assert l.gfd_kv_attend(h, bytes(c), b, bytes(a), 0) == GFD_ERR_INVALID
    assert l.gfd_kv_attend_shared(h, bytes(c), b, s.starts.data_ptr(), 16, bytes(a), 0) == GFD_ERR_INVALID
    assert l.gfd_kv_attend_workspace(h, bytes(c), b, bytes(a), 0, ctypes.byref(n)) == GFD_ERR_INVALID
    assert l.gfd_kv_append(h, bytes(c), b, bytes(kv._Append()), 0) == GFD_ERR_INVALID
    torch_().cuda.synchronize()
    assert bool((out == 7).all())


def test_a_cache_without_heads_is_refused(gpu_ctx):
    """The same through the Python layer, whose tensors may have a dimension of nothing."""
    torch = torch_()
    s = Setup(gpu_ctx, "bf16", 2, 2, 64, 16, [1, 1], [20, 30], seed=65)
    cache = kv.PagedCache(gpu_ctx, s.k[:, :, :0], s.v[:, :, :0])
    with pytest.raises(GfdError) as e:
        cache.attend(s.batch, s.q, torch.empty_like(s.q), workspace=s.workspace(1))
    assert e.value.code == GFD_ERR_INVALID
    with pytest.raises(GfdError):
        cache.append(s.batch, s.normal(2, 0, 64), s.normal(2, 0, 64))


@pytest.mark.parametrize("shared_len", [0, 100])
def test_workspace_of_the_largest_batch_serves_smaller_ones(gpu_ctx, shared_len):
    """Sequences that all have many rows, then the same program's batches with short ones among them."""
    ws = None
    for q_lens in ([90] * 4, [90, 1, 2, 90], [1] * 4, [90, 90], [3]):
        s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, q_lens, [n + 30 for n in q_lens], seed=66, shared_len=shared_len)
        if ws is None:
            ws = s.workspace(90)
        s.check(max_q_len=90, workspace=ws)


@pytest.mark.parametrize("kw", [{}, dict(softcap=3.0), dict(softcap=50.0, window=40), dict(window=40)])
@pytest.mark.parametrize("dtype,d,q_lens,kv_lens,shared", [
    ("bf16", 64, [1, 4], [45, 300], 0), ("fp16", 128, [3, 2], [500, 33], 0), ("bf16", 128, [150, 70], [200, 700], 0),
    ("fp16", 64, [200, 33], [400, 33], 0), ("bf16", 64, [2, 3, 1], [20, 40, 9], 300), ("bf16", 128, [1, 100], [9, 130], 150)])
def test_attend_bits_do_not_depend_on_what_a_row_does_not_see(gpu_ctx, dtype, d, q_lens, kv_lens, shared, kw):
    """Large keys and values where a row's mask hides them, and other rows' queries, leave every bit of it as it was."""
    torch = torch_()
    s = Setup(gpu_ctx, dtype, 2, 4, d, 16, q_lens, kv_lens, seed=67, shared_len=shared)
    a, la = s.attend(out_dtype="fp32", **kw)
    first = lambda i: max(0, kv_lens[i] - q_lens[i] - 39) if kw.get("window") else 0  # first own key that any row sees
    for i, n in enumerate(kv_lens):
        for j in list(range(first(i))) + [n - 1] + list(range(n, -(-n // 16) * 16)):  # the last key: the last row's alone
            block, place = int(s.table[i, j // 16]), j % 16
            s.k[block, place] *= 3000
            s.v[block, place] *= 30
    b, lb = s.attend(out_dtype="fp32", **kw)
    ends = [x - 1 for x in s.row_start[1:]]
    rows = [r for r in range(s.rows) if r not in ends]
    torch.cuda.synchronize()
    assert torch.equal(a[rows], b[rows]) and torch.equal(la[rows], lb[rows])
    s.q[ends] *= 40
    s.q[rows[::3]] *= 40
    c, lc = s.attend(out_dtype="fp32", **kw)
    rest = [r for r in rows if r not in rows[::3]]
    torch.cuda.synchronize()
    assert torch.equal(a[rest], c[rest]) and torch.equal(la[rest], lc[rest])


@pytest.mark.parametrize("poison", [NAN, INF])
@pytest.mark.parametrize("dtype,heads,group,d,rows,keys,kw", [
    ("bf16", 1, 2, 64, 300, 200000, {}), ("fp16", 1, 4, 128, 40, 150000, dict(window=90000)),
    ("bf16", 2, 3, 128, 20, 60000, dict(softcap=30.0, alibi=True)), ("fp16", 2, 4, 64, 4, 300000, {})])
def test_attend_masked_nan_in_a_long_context(gpu_ctx, dtype, heads, group, d, rows, keys, kw, poison):
    """The last keys, which only the last rows see, hold NaN or infinities: the other rows are summed as without
    them, in a time of the same order, and no wait runs out."""
    torch = torch_()
    s = Setup(gpu_ctx, dtype, heads, group, d, 64, [rows], [keys], seed=68)
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi"] = s.slopes()
    want = s.want(**kw)
    out, ws = torch.empty(rows, s.hq, d, device="cuda", dtype=s.dt), s.workspace(rows)
    a, b, c = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    s.attend(out=out, workspace=ws, **kw)
    a.record()
    s.attend(out=out, workspace=ws, **kw)
    b.record()
    torch.cuda.synchronize()
    n = max(1, rows // 10)
    for j in range(keys - n, keys):
        put(s, 0, j, slice(None), poison)
    b.record()
    got, lse = s.attend(out=out, workspace=ws, **kw)
    c.record()
    torch.cuda.synchronize()
    assert int(s.status) == 0
    oracle.check_attend(got, lse, want, slice(0, rows - n))
    assert not bool(torch.isfinite(got[rows - n:].float()).any())
    assert bool(torch.isfinite(lse).all())
    assert b.elapsed_time(c) < 200  # ms; without the NaN the calls take about one


@pytest.mark.parametrize("d", [64, 128])
def test_attend_mixed_units_with_and_without_nan(gpu_ctx, d):
    """Units of one stretch: some met a masked NaN, some an infinity that rows see, most nothing of the kind."""
    torch = torch_()
    q_lens = [90, 3, 200, 64, 1, 130, 70, 300]
    kv_lens = [100, 40, 700, 64, 90, 1000, 200, 300]
    s = Setup(gpu_ctx, "fp16", 8, 4, d, 16, q_lens, kv_lens, seed=69)
    want = s.want()
    ends = [b - 1 for b in s.row_start[1:]]
    for i in (0, 3, 5, 7):
        put(s, i, kv_lens[i] - 1, slice(None), NAN)
    at = kv_lens[2] - 100
    put(s, 2, at, 7, INF)
    got, lse = s.attend()
    torch.cuda.synchronize()
    assert int(s.status) == 0
    inf_rows = [s.row_start[2] + r for r in range(200) if kv_lens[2] - 200 + r >= at]
    bad = {ends[i] for i in (0, 3, 5, 7)}
    rows = [r for r in range(s.rows) if r not in bad]
    cut = lambda x, e: x[:, :, e] if x.dim() == 3 else x
    keep = [e for e in range(d) if e != 7]
    oracle.check_attend(got[:, :, keep], lse, tuple(cut(x, keep) for x in want), rows)
    oracle.check_attend(got[:, :, 7:8], lse, tuple(cut(x, [7]) for x in want), [r for r in rows if r not in set(inf_rows)])
    assert bool((got[inf_rows][:, :, 7] == INF).all()) and bool(torch.isnan(got[sorted(bad)].float()).all())


@pytest.mark.parametrize("kw", [{}, dict(softcap=20.0)])
@pytest.mark.parametrize("d,out_dtype", [(64, "fp32"), (128, None)])
def test_shared_masked_nan(gpu_ctx, d, out_dtype, kw):
    """A shared prefix whose first keys a window hides from most rows, and own keys that only the last rows see, hold NaN."""
    torch = torch_()
    q_lens, kv_lens = [1, 3, 90, 1, 200], [30, 12, 95, 1, 260]
    s = Setup(gpu_ctx, "bf16", 2, 4, d, 16, q_lens, kv_lens, seed=70, shared_len=600)
    window = 400
    want = s.want(window=window, **kw)
    first = [600 + n - m + i - window + 1 for n, m in zip(kv_lens, q_lens) for i in range(m)]
    j = min(first) + 2
    s.v[int(s.shared_table[j // 16]), j % 16] = NAN
    for i in (1, 2, 4):
        put(s, i, kv_lens[i] - 1, slice(None), INF)
    got, lse = s.attend(out_dtype=out_dtype, window=window, **kw)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    ends = [s.row_start[i + 1] - 1 for i in (1, 2, 4)]
    nan = [r for r, f in enumerate(first) if f <= j]
    rows = [r for r in range(s.rows) if r not in set(ends) | set(nan)]
    assert nan and rows
    oracle.check_attend(got, lse, want, rows)
    assert bool(torch.isnan(got[nan].float()).all()) and not bool(torch.isfinite(got[ends].float()).any())


def test_attend_padding_is_not_reported(gpu_ctx):
    """Empty sequences, whatever their lengths and tables say, a batch of none and a call of no rows: no status, nothing written."""
    torch = torch_()
    q_lens, kv_lens = [0, 90, 0, 0, 1, 0, 3, 0], [0, 90, 0, 0, 50, 0, 64, 0]
    for shared_len in (0, 40):
        s = Setup(gpu_ctx, "bf16", 2, 4, 128, 16, q_lens, kv_lens, seed=71, spare_rows=9, shared_len=shared_len)
        empty = [i for i, n in enumerate(q_lens) if n == 0]
        s.lens[empty] = torch.tensor([0, -5, 10 ** 9, 7, 1], dtype=torch.int32, device="cuda")
        s.table[empty] = -1
        s.check()
        st = torch.cuda.current_stream()
        none = kv.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), s.lens[:0], s.table[:0])
        out, ws = torch.full_like(s.q, 7.0), s.workspace()
        for batch, q, o in ((none, s.q, out), (s.batch, s.q[:0], out[:0])):
            if shared_len:
                s.cache.attend_shared(batch, s.shared_table, shared_len, q, o, workspace=ws, status=s.status, stream=st)
            else:
                s.cache.attend(batch, q, o, workspace=ws, status=s.status, stream=st)
        torch.cuda.synchronize()
        assert bool((out == 7).all()) and int(s.status) == 0


@pytest.mark.parametrize("part,out,n,rows,heads,d", [("bf16", "bf16", 2, 4099, 11, 128), ("fp32", "fp16", 3, 2999, 29, 64),
                                                     ("fp16", "fp32", 5, 5003, 8, 128)])
def test_merge_more_rows_than_threads(gpu_ctx, part, out, n, rows, heads, d):
    """So many rows and heads that a thread takes several."""
    torch = torch_()
    assert rows * heads > 16 * torch.cuda.get_device_properties(0).multi_processor_count * 256 // (d // 8)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    parts = torch.randn(n, rows, heads, d, generator=gen, device="cuda").to(types()[part])
    lse = torch.randn(n, rows, heads, generator=gen, device="cuda") * 10
    lse[1:, ::7] = float("-inf")
    lse[:, ::11] = float("-inf")
    o = torch.full((rows, heads, d), 7.0, device="cuda", dtype=types()[out])
    l = torch.full((rows, heads), 7.0, device="cuda")
    kv.merge(gpu_ctx, parts, lse, o, lse=l, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    want, wl_, tol, ltol = oracle.merge(parts, lse, types()[out])
    oracle.check_rounded(o, want, tol)
    none = torch.isinf(wl_)
    assert torch.equal(l.double()[none], wl_[none]) and bool((o[none] == 0).all())
    assert bool(((l.double() - wl_)[~none].abs() <= ltol[~none]).all())


@pytest.mark.parametrize("window", [1, 5, 60])
@pytest.mark.parametrize("d,q_lens,kv_lens", [(64, [1, 2, 1], [70, 90, 65]), (128, [1, 2, 1], [70, 90, 65]), (64, [70, 1], [140, 61]),
                                              (128, [300, 3], [400, 64])])
def test_shared_prefix_hidden_by_the_window(gpu_ctx, d, q_lens, kv_lens, window):
    """A window that ends before the shared prefix: its blocks are not looked at, not even their ids."""
    torch = torch_()
    s = Setup(gpu_ctx, "fp16", 2, 4, d, 16, q_lens, kv_lens, seed=72, spare_rows=1, shared_len=200)
    s.check(window=window)
    s.check(window=window, softcap=20.0, alibi=s.slopes())
    want = s.want(window=window)
    s.shared_table[:] = -1
    got, lse = s.attend(window=window)
    torch.cuda.synchronize()
    oracle.check_attend(got, lse, want, slice(0, s.row_start[-1]))
    assert int(s.status) == 0


@pytest.mark.parametrize("shared_len", [100, 1000])
def test_shared_blocks_that_no_row_sees_may_be_gone(gpu_ctx, shared_len):
    """Ids between what a prefix mask and what a window lets the batch see are not looked at; those that some row sees are."""
    torch = torch_()
    q_lens, kv_lens, window = [1, 2, 0, 90], [30, 40, 5, 95], 50
    s = Setup(gpu_ctx, "bf16", 2, 4, 64, 16, q_lens, kv_lens, seed=73, shared_len=shared_len)
    pre = s.ints([20, 3, 10 ** 6, -7])
    want = s.want(window=window, prefix_len=pre)
    first = min(shared_len + n - m - window + 1 for n, m in zip(kv_lens, q_lens) if m)
    kept = s.shared_table.clone()
    s.shared_table[2:first // 16] = -1
    got, lse = s.attend(window=window, prefix_len=pre)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    oracle.check_attend(got, lse, want)
    s.shared_table.copy_(kept)
    s.shared_table[first // 16] = 2 ** 31 - 1
    want = s.want(window=window, prefix_len=pre)
    got, lse = s.attend(window=window, prefix_len=pre)
    torch.cuda.synchronize()
    assert int(s.status) == kv.BAD_PAGE
    oracle.check_attend(got, lse, want)
