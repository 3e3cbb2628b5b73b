"""Cases of the paged KV-cache operators and how each is run.

The four operators work on blocks of the kind the library fetches from host memory
(block = tokens x KV heads x head dim of K, then of V): append (with the rotation of
positions), attend, attend over a shared prefix, and merge of partial results.

`listed()` and `draw()` give cases, `prepare()` makes what a program has in hand before
the call, `run()` makes one pass: with the module's `own` false in elementary torch
operations in 32 bits (angles in 64), with `own` true through gfd_b200.kv.
`exact()` computes the same outputs in 64 bits from the definitions.

Positions: sequence s has kv_len[s] tokens in the cache, the last q_len[s] of them being
the call's own rows, so row i stands at position p = kv_len[s] - q_len[s] + i (behind a
shared prefix of P tokens: P more).  Row p sees key j when

    j < prefix_len[s]  or  ((not causal or j <= p) and (window == 0 or j > p - window))

and its scores are  cap * tanh(scale * q.k / cap) + slope[head] * (j - p)  (each part only
where the case has it).  A row that sees nothing gives zeros, and lse = -inf.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _paged(**kw):
    """A case of append / attend / shared: the values a case does not name."""
    case = dict(dtype="bf16", seqs=1, lead_q=0, q_min=1, q_max=1, hist_min=0, hist_max=0, lens=1, q_heads=32,
                kv_heads=8, head_dim=128, block_tokens=16, blocks=0)
    if kw["op"] == "append":
        case.update(rot_dim=128, interleaved=False)
    else:
        case.update(causal=True, window=0, prefix=0, softcap=0.0, alibi=False)
    if kw["op"] == "shared":
        case.update(shared_len=0)
    case.update(kw)
    return case


def listed():
    return [
        # one decode step of a small batch: 8 tokens into 64 KiB blocks of 16 tokens; the
        # smallest append, where only latency counts
        _paged(name="append_decode", op="append", seqs=8, hist_max=4000, lens=11),
        # prompt chunks of three requests, pairs of neighbouring elements rotated and only
        # half of each head, larger blocks
        _paged(name="append_prompt", op="append", dtype="fp16", seqs=3, q_min=1800, q_max=4001, hist_max=700, lens=12,
               block_tokens=64, rot_dim=64, interleaved=True),
        # a decode step far into long contexts (positions near a million): the angles need
        # more than 32 bits; one KV head, seven query heads
        _paged(name="append_far", op="append", seqs=33, hist_min=400000, hist_max=1000000, lens=13, q_heads=7, kv_heads=1,
               head_dim=64, rot_dim=64),
        # one user, one token, a short context: latency
        _paged(name="attend_one", op="attend", hist_min=776, hist_max=776, lens=21),
        # the decode step of a serving batch over a 4 GiB pool of 64 KiB blocks, lengths spread
        # from short to long: the reading of the cache
        _paged(name="attend_batch", op="attend", seqs=64, hist_min=100, hist_max=8191, lens=22, blocks=65536),
        # two long contexts, capped scores and a bias that falls with the distance
        _paged(name="attend_long", op="attend", dtype="fp16", seqs=2, hist_min=120000, hist_max=131071, lens=23, q_heads=24,
               head_dim=64, block_tokens=32, softcap=50.0, alibi=True),
        # two whole prompts, causal: the matrix products
        _paged(name="attend_prompt", op="attend", seqs=2, q_min=5000, q_max=8191, lens=24),
        # a chunk of one prompt among decoding requests; a sliding window beside a prefix that
        # every row sees, capped scores
        _paged(name="attend_mixed", op="attend", dtype="fp16", seqs=32, lead_q=2048, hist_min=50, hist_max=9000, lens=25,
               q_heads=14, kv_heads=2, head_dim=64, window=4096, prefix=100, softcap=30.0),
        # 64 requests behind one long system prompt, own contexts short
        _paged(name="shared_batch", op="shared", seqs=64, hist_max=512, lens=31, shared_len=16384),
        # a few requests that verify three drafted tokens each behind a short common prompt
        _paged(name="shared_few", op="shared", dtype="fp16", seqs=7, q_min=3, q_max=3, hist_max=90, lens=32, q_heads=20,
               kv_heads=4, head_dim=64, shared_len=1111),
        # resident and fetched part of a decode batch joined
        dict(name="merge_decode", op="merge", dtype="bf16", part_dtype="bf16", parts=2, tokens=64, heads=32, head_dim=128),
        # a prompt's rows joined from four parts that were kept in 32 bits
        dict(name="merge_prompt", op="merge", dtype="bf16", part_dtype="fp32", parts=4, tokens=8191, heads=32, head_dim=128),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:  # within the cost of the largest listed cases
        case = _draw(rng)
        cost = work(case)
        if cost["bytes"] < 1.0e9 and cost["flops"] < 6.0e11:
            return case


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "shared", "merge"])
    dtype = rng.choice(["bf16", "fp16"])
    head_dim = rng.choice([64, 128])
    lens = rng.randrange(1, 1 << 30)
    if op == "merge":
        heads = rng.randint(1, 40)
        return dict(op=op, dtype=dtype, part_dtype=rng.choice([dtype, "fp32"]), parts=rng.randint(2, 8),
                    tokens=_spread(rng, 1, 32768 // heads), heads=heads, head_dim=head_dim)
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    case = _paged(op=op, dtype=dtype, lens=lens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                  block_tokens=rng.choice([16, 16, 32, 64]))
    if op == "append":
        seqs = _spread(rng, 1, 128)
        q = _spread(rng, 1, 8192 // seqs)
        case.update(seqs=seqs, q_min=max(1, q // 2), q_max=q, hist_max=_spread(rng, 1, 100000),
                    rot_dim=rng.choice([0, 32, 64, head_dim]), interleaved=rng.random() < 0.5)
        return case
    case.update(softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.25)
    if op == "shared":
        seqs = _spread(rng, 2, 100)
        case.update(seqs=seqs, q_max=rng.choice([1, 1, 2, 5]), hist_max=_spread(rng, 1, 1000),
                    shared_len=_spread(rng, 17, 20000), window=rng.choice([0, 0, 0, 5000]))
        return case
    kind = rng.choice(["decode", "prompt", "mixed"])
    if kind == "decode":
        seqs = _spread(rng, 1, 100)
        case.update(seqs=seqs, hist_max=_spread(rng, 1, min(130000, 400000 // seqs)))
    elif kind == "prompt":
        seqs = rng.randint(1, 4)
        q = _spread(rng, 2, 8000 // seqs)
        case.update(seqs=seqs, q_min=max(1, q // 2), q_max=q, hist_max=_spread(rng, 1, 2000), causal=rng.random() < 0.8)
    else:
        case.update(seqs=_spread(rng, 2, 40), lead_q=_spread(rng, 16, 2500), q_max=rng.choice([1, 1, 4]),
                    hist_max=_spread(rng, 1, 9000))
    case.update(window=rng.choice([0, 0, _spread(rng, 16, 4096)]), prefix=rng.choice([0, 0, _spread(rng, 1, 300)]))
    return case


def lengths(case):
    """(q_len, kv_len) of every sequence, from the case alone."""
    rng = random.Random(case["lens"])
    q = [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    if case["lead_q"]:
        q[0] = case["lead_q"]
    return q, [n + rng.randint(case["hist_min"], case["hist_max"]) for n in q]


def _spans(case, q_len, kv_len, device="cpu"):
    """Per row of one sequence: position p and the visible keys [0, pre) and [lo, hi)."""
    shift = case.get("shared_len", 0)
    n = shift + kv_len
    p = torch.arange(q_len, dtype=torch.int64, device=device) + (n - q_len)
    pre = torch.full_like(p, min(case["prefix"], n))
    hi = torch.clamp(p + 1, max=n) if case["causal"] else torch.full_like(p, n)
    lo = torch.clamp(p + 1 - case["window"], min=0) if case["window"] else torch.zeros_like(p)
    return p, pre, lo, hi


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "merge":
        n = case["tokens"] * case["heads"]
        part = 4 if case["part_dtype"] == "fp32" else 2
        return {"bytes": case["parts"] * n * (case["head_dim"] * part + 4) + n * (case["head_dim"] * 2 + 4),
                "flops": 2 * case["parts"] * n * case["head_dim"]}
    q, kv = lengths(case)
    d, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        # k, v and q are read once and written once
        rows = sum(q)
        return {"bytes": rows * d * 2 * 2 * (2 * hkv + hq), "flops": rows * 3 * case["rot_dim"] * (hq + hkv)}
    pairs, keys, shared = 0, 0, case.get("shared_len", 0)
    shared_lo = shared
    for ql, kl in zip(q, kv):
        _, pre, lo, hi = _spans(case, ql, kl)
        both = torch.clamp(torch.minimum(pre, hi) - lo, min=0)
        pairs += int((torch.clamp(hi - lo, min=0) + pre - both).sum())
        # the keys that any of its rows sees, those of the shared prefix apart
        first, last, pre0 = int(lo[0]), int(hi[-1]), int(pre[0])
        keys += max(0, last - max(shared, first, pre0)) + max(0, pre0 - shared)
        shared_lo = min(shared_lo, first)
    keys += shared - shared_lo
    return {"bytes": keys * hkv * d * 2 * 2 + sum(q) * hq * (2 * d * 2 + 4), "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _table(case, kv, q, gen):
    """Block table: the blocks that hold the call's own rows are distinct, the others are
    drawn from what is left (a pool smaller than the contexts repeats them)."""
    bt = case["block_tokens"]
    width = max((n + bt - 1) // bt for n in kv) or 1
    need = sum((n + bt - 1) // bt for n in kv)
    fresh = sum((n + bt - 1) // bt - (n - m) // bt for n, m in zip(kv, q))
    blocks = case["blocks"] or (fresh + 64 if case["op"] == "append" else need + 3)
    perm = torch.randperm(blocks, generator=gen, device="cuda", dtype=torch.int64).tolist()
    mine, rest = perm[:fresh], perm[fresh:]
    mine, rest = torch.tensor(mine, dtype=torch.int32), torch.tensor(rest, dtype=torch.int32)
    table = torch.zeros(len(kv), width, dtype=torch.int32)
    at = used = 0
    for s, (n, m) in enumerate(zip(kv, q)):
        total = (n + bt - 1) // bt
        new = total - (n - m) // bt
        old = total - new
        table[s, :old] = rest[torch.arange(used, used + old) % len(rest)]
        table[s, old:total] = mine[at:at + new]
        used += old
        at += new
    return table.cuda(), blocks


_contexts = {}


def _context():
    """The library's handle of the current GPU: a program makes one and keeps it."""
    import gfd_b200
    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = gfd_b200.Context(device)
    return _contexts[device]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    d = case["head_dim"]
    state = {"case": case}
    if case["op"] == "merge":
        t, h = case["tokens"], case["heads"]
        state["parts"] = normal(case["parts"], t, h, d, dtype=TYPES[case["part_dtype"]])
        state["part_lse"] = normal(case["parts"], t, h, dtype=torch.float32) * 2 + 5
        state["out"] = torch.empty(t, h, d, device="cuda", dtype=dt)
        state["lse"] = torch.empty(t, h, device="cuda", dtype=torch.float32)
        if own:
            state["ctx"] = _context()
        return state
    q, kv = lengths(case)
    hq, hkv, bt = case["q_heads"], case["kv_heads"], case["block_tokens"]
    shared_blocks = (case.get("shared_len", 0) + bt - 1) // bt
    table, blocks = _table(case, kv, q, gen)
    # one block: K of its tokens, then V of its tokens
    pool = normal(blocks + shared_blocks, 2, bt, hkv, d)
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    state.update(q_len=q, kv=kv, pool=pool, table=table, q=normal(rows, hq, d) * 2,
                 q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 kv_len=torch.tensor(kv, dtype=torch.int32, device="cuda"))
    if case["op"] == "append":
        state.update(k=normal(rows, hkv, d), v=normal(rows, hkv, d), q_out=torch.empty(rows, hq, d, device="cuda", dtype=dt))
        r = case["rot_dim"]
        state["inv_freq"] = torch.tensor([10000.0 ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float32,
                                         device="cuda") if r else None
    else:
        state["out"] = torch.empty(rows, hq, d, device="cuda", dtype=dt)
        state["lse"] = torch.empty(rows, hq, device="cuda", dtype=torch.float32)
        state["alibi"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32,
                                      device="cuda") if case["alibi"] else None
        state["prefix_len"] = torch.full((len(q),), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        if case["op"] == "shared":
            state["shared_table"] = torch.randperm(shared_blocks, generator=gen, device="cuda").to(torch.int32) + blocks
    if own:
        from gfd_b200 import kv as gkv
        state["ctx"] = _context()
        state["cache"] = gkv.PagedCache(state["ctx"], pool[:, 0], pool[:, 1])
        state["batch"] = gkv.Batch(state["q_start"], state["kv_len"], table)
        if case["op"] != "append":
            nbytes = state["cache"].workspace_bytes(rows, hq, seqs=len(q), max_q_len=max(q),
                                                    shared_len=case.get("shared_len", 0))
            state["workspace"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "shared": _plain_attend, "merge": _plain_merge}[op](state)


def _run_own(st):
    case = st["case"]
    stream = torch.cuda.current_stream()
    if case["op"] == "merge":
        from gfd_b200 import kv as gkv
        gkv.merge(st["ctx"], st["parts"], st["part_lse"], st["out"], lse=st["lse"], stream=stream)
        return [st["out"], st["lse"]]
    if case["op"] == "append":
        st["cache"].append(st["batch"], st["k"], st["v"], q=st["q"], q_out=st["q_out"], inv_freq=st["inv_freq"],
                           interleaved=case["interleaved"], stream=stream)
        return [st["q_out"], st["pool"]]
    kw = dict(lse=st["lse"], scale=case["head_dim"] ** -0.5, causal=case["causal"], window=case["window"],
              softcap=case["softcap"], alibi=st["alibi"], prefix_len=st["prefix_len"], max_q_len=max(st["q_len"]),
              workspace=st["workspace"], stream=stream)
    if case["op"] == "shared":
        st["cache"].attend_shared(st["batch"], st["shared_table"], case["shared_len"], st["q"], st["out"], **kw)
    else:
        st["cache"].attend(st["batch"], st["q"], st["out"], **kw)
    return [st["out"], st["lse"]]


def _rotate(x, cos, sin, interleaved):
    """x [rows, heads, d] with its first 2 * cos.shape[1] elements rotated."""
    half = cos.shape[1]
    if half == 0:
        return x
    cos, sin = cos[:, None, :], sin[:, None, :]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_append(st):
    case, dt = st["case"], st["q"].dtype
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(st["q_len"], st["kv"])])
    seq = torch.cat([torch.full((m,), s, device="cuda", dtype=torch.int64) for s, m in enumerate(st["q_len"])])
    freq = st["inv_freq"].double() if case["rot_dim"] else torch.zeros(0, dtype=torch.float64, device="cuda")
    angle = pos.double()[:, None] * freq[None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    bt = case["block_tokens"]
    block = st["table"][seq, pos // bt].long()
    st["pool"][block, 0, pos % bt] = _rotate(st["k"].float(), cos, sin, case["interleaved"]).to(dt)
    st["pool"][block, 1, pos % bt] = st["v"]
    st["q_out"].copy_(_rotate(st["q"].float(), cos, sin, case["interleaved"]).to(dt))
    return [st["q_out"], st["pool"]]


def _dense(st, s):
    """K and V of sequence s [kv_heads, keys, d], the shared prefix in front."""
    bt, n = st["case"]["block_tokens"], st["kv"][s]
    blocks = st["pool"][st["table"][s, :(n + bt - 1) // bt].long()]
    k, v = blocks[:, 0].flatten(0, 1)[:n], blocks[:, 1].flatten(0, 1)[:n]
    if "shared_table" in st:
        pre = st["pool"][st["shared_table"].long()]
        p = st["case"]["shared_len"]
        k = torch.cat([pre[:, 0].flatten(0, 1)[:p], k])
        v = torch.cat([pre[:, 1].flatten(0, 1)[:p], v])
    return k.transpose(0, 1), v.transpose(0, 1)


def _plain_attend(st):
    case = st["case"]
    scale, group = case["head_dim"] ** -0.5, case["q_heads"] // case["kv_heads"]
    row0 = 0
    for s, (ql, kl) in enumerate(zip(st["q_len"], st["kv"])):
        k, v = _dense(st, s)
        k, v = k.float(), v.float()
        n = k.shape[1]
        p, pre, lo, hi = _spans(case, ql, kl, "cuda")
        j = torch.arange(n, device="cuda")
        step = max(1, (1 << 28) // max(1, n * case["q_heads"]))
        for a in range(0, ql, step):
            b = min(ql, a + step)
            x = st["q"][row0 + a:row0 + b].float()  # [rows, q_heads, d]
            x = x.view(b - a, case["kv_heads"], group, -1).permute(1, 2, 0, 3).flatten(1, 2)
            z = (x @ k.transpose(1, 2)).view(case["kv_heads"], group, b - a, n) * scale
            if case["softcap"]:
                z = torch.tanh(z / case["softcap"]) * case["softcap"]
            if case["alibi"]:
                dist = (j[None, :] - p[a:b, None]).float()
                z = z + st["alibi"].view(case["kv_heads"], group, 1, 1) * dist
            seen = (j < pre[a:b, None]) | ((j >= lo[a:b, None]) & (j < hi[a:b, None]))
            z = torch.where(seen, z, torch.full_like(z, float("-inf")))
            m = z.amax(-1, keepdim=True)
            m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
            e = torch.exp(z - m)
            total = e.sum(-1, keepdim=True)
            o = (e.flatten(1, 2) @ v).view(case["kv_heads"], group, b - a, -1)
            o = torch.where(total > 0, o / total, torch.zeros_like(o))
            st["out"][row0 + a:row0 + b] = o.permute(2, 0, 1, 3).flatten(1, 2).to(st["out"].dtype)
            st["lse"][row0 + a:row0 + b] = (torch.log(total) + m)[..., 0].permute(2, 0, 1).flatten(1, 2)
        row0 += ql
    return [st["out"], st["lse"]]


def _plain_merge(st):
    lse = st["part_lse"]
    m = lse.amax(0)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    w = torch.exp(lse - m)
    total = w.sum(0)
    out = (st["parts"].float() * w[..., None]).sum(0)
    out = torch.where(total[..., None] > 0, out / total[..., None], torch.zeros_like(out))
    st["out"].copy_(out.to(st["out"].dtype))
    st["lse"].copy_(torch.log(total) + m)
    return [st["out"], st["lse"]]


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"append": _exact_append, "attend": _exact_attend, "shared": _exact_attend, "merge": _exact_merge}[case["op"]](st)


def _exact_append(st):
    case = st["case"]
    half, d, bt = case["rot_dim"] // 2, case["head_dim"], case["block_tokens"]
    # pair i of a head: elements first[i] and second[i]
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    pool = st["pool"].double()
    q_out = st["q"].double()
    freq = st["inv_freq"].double() if half else None
    row = 0
    for s, (m, n) in enumerate(zip(st["q_len"], st["kv"])):
        pos = torch.arange(n - m, n, device="cuda")
        k = st["k"][row:row + m].double()
        if half:
            turn = torch.polar(torch.ones(m, half, dtype=torch.float64, device="cuda"), torch.outer(pos.double(), freq))
            for x in (k, q_out[row:row + m]):
                z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
                x[..., first], x[..., second] = z.real, z.imag
        ids = st["table"][s].long()[torch.div(pos, bt, rounding_mode="floor")]
        pool[ids, 0, pos % bt] = k
        pool[ids, 1, pos % bt] = st["v"][row:row + m].double()
        row += m
    return [q_out, pool]


def _exact_attend(st):
    case = st["case"]
    hq, group, d = case["q_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    base = 0
    for s, (ql, kl) in enumerate(zip(st["q_len"], st["kv"])):
        keys, vals = _dense(st, s)
        n = keys.shape[1]
        at = torch.arange(n, device="cuda")[None, :]
        for h in range(hq):
            kh, vh = keys[h // group].double(), vals[h // group].double()
            step = max(1, (1 << 26) // max(1, n))
            for a in range(0, ql, step):
                b = min(ql, a + step)
                here = torch.arange(a, b, device="cuda")[:, None] + (n - ql)
                x = torch.einsum("rd,nd->rn", st["q"][base + a:base + b, h].double(), kh) / math.sqrt(d)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                if case["alibi"]:
                    x = x - float(st["alibi"][h]) * (here - at).double()
                hidden = torch.zeros(b - a, n, dtype=torch.bool, device="cuda")
                if case["causal"]:
                    hidden |= at > here
                if case["window"]:
                    hidden |= here - at >= case["window"]
                if case["prefix"]:
                    hidden &= at >= case["prefix"]
                x = x.masked_fill(hidden, float("-inf"))
                l = torch.logsumexp(x, 1)
                w = torch.exp(x - torch.where(torch.isinf(l), torch.zeros_like(l), l)[:, None])
                out[base + a:base + b, h] = torch.einsum("rn,nd->rd", w, vh)
                lse[base + a:base + b, h] = l
        base += ql
    return [out, lse]


def _exact_merge(st):
    lse = torch.logsumexp(st["part_lse"].double(), 0)
    safe = torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    for part, l in zip(st["parts"], st["part_lse"]):
        out += part.double() * torch.exp(l.double() - safe)[..., None]
    return [out, lse]
