"""Rotary positions, the append to a paged int8 cache and the attention over it, from their formulas in float64 on the CPU, and the inputs
that their tests share."""
import math

import torch

LEAST_SCALE = 2.0 ** -100


def rotate(x, positions, freqs, magnitude=1.0, interleaved=False, inverse=False):
    """x [Z, H, N, d], positions [Z, N]; float64."""
    x = x.double()
    pairs = freqs.numel()
    angle = positions.double()[:, None, :, None] * freqs.double()
    c, s = angle.cos() * magnitude, angle.sin() * magnitude * (-1.0 if inverse else 1.0)
    y = x.clone()
    even, odd = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., even], x[..., odd]
    y[..., even], y[..., odd] = a * c - b * s, b * c + a * s
    return y


def finite(x):
    """Values that count for a page's scale, and what is quantised in the place of the others."""
    return torch.where(torch.isfinite(x), x, torch.zeros_like(x))


def append(cache, scale, rows, table, lens, fresh):
    """rows [Z, H, N, d] in fp32 into cache [pages, H, page, d] int8 and scale [pages, H] fp32, in place, in the kernel's fp32 steps."""
    pages, H, page, d = cache.shape
    for z in range(rows.shape[0]):
        n, m = max(0, int(lens[z])), max(0, min(int(fresh[z]), rows.shape[2]))
        at = n
        while at < n + m and at // page < table.shape[1]:
            r = at % page
            k = min(page - r, n + m - at)
            p = int(table[z, at // page])
            if 0 <= p < pages:
                new = rows[z, :, at - n:at - n + k].float()
                s = torch.clamp(finite(new).abs().amax((-1, -2)) / torch.tensor(127.0), min=LEAST_SCALE)
                if r > 0:
                    s = torch.maximum(s, scale[p])
                    ratio = scale[p] / s
                    cache[p, :, :r] = torch.where((s != scale[p])[:, None, None],
                                                  torch.round(cache[p, :, :r].float() * ratio[:, None, None]).to(torch.int8), cache[p, :, :r])
                q = torch.nan_to_num(torch.round(new / s[:, None, None]), nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127)
                cache[p, :, r:r + k] = q.to(torch.int8)
                scale[p] = s
            at += k


def attend(q, cache, table, lens, causal, sm, fresh=None, rope=None):
    """q [Z, H, N, d]; cache: dict of k, v [pages, H_kv, page, d] and ks, vs [pages, H_kv].  Returns the output, lse (base 2), and for the bound on
    errors the mean of |v| under the row's weights and the largest sum of |q k| of a visible key."""
    Z, H, N, d = q.shape
    pages, Hkv, page, _ = cache["k"].shape
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full((Z, H, N), -math.inf, dtype=torch.float64)
    mean_v, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros((Z, H, N, 1), dtype=torch.float64)
    for z in range(Z):
        n = max(0, min(int(lens[z]), table.shape[1] * page))
        m = N if fresh is None else max(0, min(int(fresh[z]), N))
        if n == 0 or m == 0:
            continue
        ids = table[z, :(n + page - 1) // page].long()
        there = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:n]
        ids = ids.clamp(0, pages - 1)
        k = (cache["k"][ids].double() * cache["ks"][ids].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, d)[:, :n]
        v = (cache["v"][ids].double() * cache["vs"][ids].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, d)[:, :n]
        k[:, ~there] = 0.0
        v[:, ~there] = 0.0
        place = torch.arange(n - m, n)
        x = q[z:z + 1, :, :m].double()
        if rope is not None:
            x = rotate(x, place[None], **rope)
        x = x[0].reshape(Hkv, H // Hkv, m, d)
        s = torch.einsum("hgmd,hnd->hgmn", x, k) * sm
        seen = there[None, :].expand(m, n)
        if causal:
            seen = seen & (torch.arange(n)[None, :] <= place[:, None])
        s = s.masked_fill(~seen, -math.inf)
        any_key = seen.any(-1)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp(), torch.zeros_like(s))
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(total == 0, torch.ones_like(total), total)
        out[z, :, :m] = torch.einsum("hgmn,hnd->hgmd", w, v).reshape(H, m, d)
        mean_v[z, :, :m] = torch.einsum("hgmn,hnd->hgmd", w, v.abs()).reshape(H, m, d)
        size[z, :, :m] = (torch.einsum("hgmd,hnd->hgmn", x.abs(), k.abs()) * abs(sm) * seen).amax(-1, keepdim=True).reshape(H, m, 1)
        lse[z, :, :m] = torch.where(any_key, ((top + total.log()) / math.log(2.0))[..., 0], torch.full((), -math.inf, dtype=torch.float64)).reshape(H, m)
    return out, lse, mean_v, size


def bound(out, mean_v, size, dtype, query_step=0.0):
    """How far the kernel may be from the above: half a step of the output's type; P rounded to 11 bits (half a step, 2^-11 of each weight, so at
    most 2^-11 of the mean of |v|); scores off by dS move a weight by dS and their sum as much: the products of a score are summed in
    fp32 in at most 13 roundings, scaled and exponentiated in a few more, 2^-19 of the sum of |q k| in all; sums over keys 2^-14.
    query_step: where the queries are rounded after their rotation, half a step of theirs, which moves a score by as much of the sum of |q k| (each product
    is off by at most half a step of its query's element): 2^-12 for the 11 bits that many rows of bf16 queries are held to."""
    return torch.finfo(dtype).eps / 2 * out.abs() + 1.05 * (2.0 ** -11 + 2.0 ** -14 + 2.0 * (2.0 ** -19 + query_step) * size) * mean_v + 2.0 ** -24


def make_cache(g, pages, Hkv, page, d, spread=0.0):
    """Pages whose scales differ by a factor of up to e^spread either way.  K and V lie side by side in one tensor, as views."""
    kv = (torch.randn((pages, 2, Hkv, page, d), generator=g) * 31.75).round().clamp(-127, 127).to(torch.int8)
    sc = torch.exp(spread * (2.0 * torch.rand((pages, 2, Hkv), generator=g) - 1.0)) / 31.75
    return dict(k=kv[:, 0], v=kv[:, 1], ks=sc[:, 0], vs=sc[:, 1]), kv, sc


def make_table(g, lens, page, pages, extra=0):
    """Shuffled pages of each sequence; columns behind the last one hold numbers that name no page of it (some of them not even of the pool)."""
    width = max(1, max((n + page - 1) // page for n in lens)) + extra
    table = torch.randint(-7, 2 * pages, (len(lens), width), generator=g, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    for z, n in enumerate(lens):
        used = (n + page - 1) // page
        table[z, :used] = order[at:at + used]
        at += used
    return table
