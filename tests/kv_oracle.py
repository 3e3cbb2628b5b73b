"""The paged KV-cache operators in 64 bits, row by row from their definitions, with error
bounds for results computed in 32 bits and rounded.

Bounds.  u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t.
Attention: with w_j the exact weights (sum 1) and A = sum w_j |v_j|,
  - a score's error d: products of two 16-bit values are exact in 32 bits and a sum of D of
    them errs by at most D u32 sum |q_i k_i|; scale, cap, bias and the move to base 2 round a
    value of at most Z eight times at most; a cap's tanh errs by at most 2^-20;
  - weights exp(z - m) then err relatively by d plus 2^-20 for the exponential, numerator
    and denominator alike: 2 (d + 2^-20) A;
  - weights rounded to the 16-bit type for the product with V: u(t) A;
  - sums over n keys in any order in 32 bits, of the numerator and the denominator:
    2 n 2^-23 A (2^-23: an accumulator that truncates);
  - the result rounds once to the output type: u(out) |o|.
"""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gather(k, v, ids, n):
    """Keys and values of n tokens in the blocks `ids` (list of (block, ok)), plus validity."""
    bt = k.shape[1]
    ids = torch.as_tensor(ids, device=k.device, dtype=torch.int64)
    ok = (ids >= 0) & (ids < k.shape[0])
    safe = torch.where(ok, ids, torch.zeros_like(ids))
    kk = k[safe].flatten(0, 1)[:n]
    vv = v[safe].flatten(0, 1)[:n]
    return kk, vv, ok.repeat_interleave(bt)[:n]


def attend(k, v, row_start, kv_len, table, q, scale, causal=True, window=0, softcap=0.0, alibi=None, prefix=None,
           shared_table=None, shared_len=0):
    """(out, lse, out bound without the output's rounding, lse bound), all [rows, ...] in 64 bits."""
    rows, hq, d = q.shape
    hkv, bt = k.shape[2], k.shape[1]
    g = hq // hkv
    dev = q.device
    out = torch.zeros(rows, hq, d, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((rows, hq), float("-inf"), dtype=torch.float64, device=dev)
    ltol = torch.zeros(rows, hq, dtype=torch.float64, device=dev)
    ut = half_step(q.dtype)
    for s in range(len(kv_len)):
        r0, r1 = row_start[s], row_start[s + 1]
        if r1 <= r0:
            continue
        n = shared_len + kv_len[s]
        kk, vv, ok = gather(k, v, table[s][:(kv_len[s] + bt - 1) // bt], kv_len[s])
        if shared_len:
            k2, v2, ok2 = gather(k, v, shared_table[:(shared_len + bt - 1) // bt], shared_len)
            kk, vv, ok = torch.cat([k2, kk]), torch.cat([v2, vv]), torch.cat([ok2, ok])
        for i in range(r1 - r0):
            p = n - (r1 - r0) + i
            j = torch.arange(n, device=dev)
            seen = torch.ones(n, dtype=torch.bool, device=dev)
            if causal:
                seen &= j <= p
            if window:
                seen &= j > p - window
            if prefix is not None:
                seen |= j < prefix[s]
            seen &= ok
            j = j[seen]
            if j.numel() == 0:
                continue
            x = q[r0 + i].double().view(hkv, g, d)
            kd, vd = kk[seen].double(), vv[seen].double()
            z = torch.einsum("hgd,nhd->hgn", x, kd) * scale
            mag = torch.einsum("hgd,nhd->hgn", x.abs(), kd.abs()) * abs(scale)
            size = mag.clone()
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if alibi is not None:
                bias = alibi.double().view(hkv, g, 1) * (j - p).double()
                z, size = z + bias, size + bias.abs()
            delta = (d * U32 * mag + 8 * U32 * size + (softcap * 2.0 ** -20 if softcap else 0)).amax(-1)
            l = torch.logsumexp(z, -1)
            w = torch.exp(z - l[..., None])
            o = torch.einsum("hgn,nhd->hgd", w, vd)
            a = torch.einsum("hgn,nhd->hgd", w, vd.abs())
            m = j.numel()
            out[r0 + i] = o.reshape(hq, d)
            lse[r0 + i] = l.reshape(hq)
            tol[r0 + i] = (a * (ut + 2 * (delta[..., None] + 2.0 ** -20) + 2 * m * 2.0 ** -23)).reshape(hq, d)
            ltol[r0 + i] = (delta + 2.0 ** -20 + m * 2.0 ** -23 + 8 * U32 * (l.abs() + z.abs().amax(-1))).reshape(hq)
    return out, lse, tol, ltol


def check_attend(got, got_lse, want, rows=None):
    out, lse, tol, ltol = want
    sel = slice(None) if rows is None else rows
    u = half_step(got.dtype)
    err = (got.double() - out)[sel].abs()
    bound = (tol * (1 + u) + u * out.abs() + 2.0 ** -25)[sel]  # 2^-25: half the smallest fp16 step
    assert not torch.isnan(got[sel].double()).any()
    assert bool((err <= bound).all()), f"out: {float((err - bound).max())} over its bound of about {float(bound.mean())}"
    if got_lse is not None:
        a, b = got_lse.double()[sel], lse[sel]
        none = torch.isinf(b)
        assert torch.equal(a[none], b[none])
        e = (a - b)[~none].abs()
        assert bool((e <= ltol[sel][~none]).all()), f"lse: off by {float(e.max())}"


def rotate(x, pos, inv_freq, interleaved):
    """x [rows, heads, d] rotated in 64 bits, and the bound of its error before the last rounding:
    sine and cosine err by at most 2^-22 (32-bit sine of a reduced angle), products and the
    sum by 3 u32."""
    half = inv_freq.shape[0]
    y = x.double().clone()
    err = torch.zeros_like(y)
    if half == 0:
        return y, err
    first = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    err[..., first] = err[..., second] = (a.abs() + b.abs()) * (2.0 ** -22 + 3 * U32)
    return y, err


def check_rounded(got, want, err):
    u = half_step(got.dtype)
    e = (got.double() - want).abs()
    bound = u * want.abs() + (1 + u) * err + 2.0 ** -25
    assert bool((e <= bound).all()), f"off by {float((e - bound).max())} over the bound"


def merge(parts, part_lse, out_dtype):
    """(out, lse, out bound, lse bound): weights err by 2^-20 for the exponential and 4 roundings of
    a difference of at most |lse|; sums of n parts by n u32."""
    lse = torch.logsumexp(part_lse.double(), 0)
    base = torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)
    out = torch.zeros(parts.shape[1:], dtype=torch.float64, device=parts.device)
    mass = torch.zeros_like(out)
    size = torch.zeros_like(lse)
    for x, l in zip(parts, part_lse):
        w = torch.exp(l.double() - base)[..., None]
        live = w > 0
        xx = torch.where(live, x.double(), torch.zeros_like(out))
        out += w * xx
        mass += w * xx.abs()
        size = torch.maximum(size, torch.where(torch.isinf(l), torch.zeros_like(base), l.double().abs()))
    rel = 2.0 ** -20 + 8 * U32 * size + 2 * parts.shape[0] * U32
    return out, lse, mass * (2 * rel)[..., None], rel + 8 * U32 * size
