"""The latent cache's append and the attention over it, and the expanded form, from their formulas in float64 on the CPU, and the inputs that their tests share."""
import math

import torch

from paged_reference import LEAST_SCALE, rotate


def normalised(c, weight, eps):
    c = c.double()
    return c / torch.sqrt(c.square().mean(-1, keepdim=True) + eps) * weight.double()


def append(cache, scale, c, k, table, lens, fresh=None, rope=None, weight=None, eps=1e-6):
    """c [Z, N, dc], k [Z, N, dr].  Returns the cache's values before their rounding where tokens are new (NaN elsewhere, float64) and the scales (float64),
    and where the new tokens are."""
    pages, page, d = cache.shape
    dc = c.shape[-1]
    values = torch.full((pages, page, d), math.nan, dtype=torch.float64)
    scales, new = scale.double().clone(), torch.zeros((pages, page), dtype=torch.bool)
    for z in range(c.shape[0]):
        n = max(0, int(lens[z]))
        m = c.shape[1] if fresh is None else max(0, min(int(fresh[z]), c.shape[1]))
        for i in range(m):
            column, r = (n + i) // page, (n + i) % page
            if column >= table.shape[1] or not 0 <= int(table[z, column]) < pages:
                continue
            p = int(table[z, column])
            x = c[z, i].double() if weight is None else normalised(c[z, i], weight, eps)
            y = k[z, i].double()
            if rope is not None:
                y = rotate(y[None, None, None], torch.tensor([[n + i]]), **rope)[0, 0, 0]
            new[p, r] = True
            for part, v in enumerate((x, y)):
                finite = torch.where(torch.isfinite(v) & (v.abs() < 3.5e38), v, torch.zeros_like(v))
                scales[p, r, part] = max(float(finite.abs().max()) / 127.0, LEAST_SCALE)
            values[p, r, :dc], values[p, r, dc:] = x, y
    return values, scales, new


def make_pool(g, pages, page, dc, dr, spread=0.0):
    cache = (torch.randn((pages, page, dc + dr), generator=g) * 31.75).round().clamp(-127, 127).to(torch.int8)
    scale = torch.exp(spread * (2.0 * torch.rand((pages, page, 2), generator=g) - 1.0)) / 31.75
    return cache, scale


def attend(q_latent, q_rope, cache, scale, table, lens, causal, sm, fresh=None, rope=None):
    """q_latent [Z, H, N, dc], q_rope [Z, H, N, dr].  Returns the output, lse (base 2), and for the bound on errors (as a part of 2^-11, the steps of weights): the mean of |v| under the row's weights and what steps of
    small weights add, the largest sum of |q k| of a visible key, and the largest error of a visible key's score that half a step of the row's queries makes."""
    Z, H, N, dc = q_latent.shape
    pages, page, _ = cache.shape
    out, lse = torch.zeros(q_latent.shape, dtype=torch.float64), torch.full((Z, H, N), -math.inf, dtype=torch.float64)
    mean_v, size, step = torch.zeros_like(out), torch.zeros((Z, H, N, 1), dtype=torch.float64), torch.zeros((Z, H, N, 1), dtype=torch.float64)
    for z in range(Z):
        n = max(0, min(int(lens[z]), table.shape[1] * page))
        m = N if fresh is None else max(0, min(int(fresh[z]), N))
        if n == 0 or m == 0:
            continue
        ids = table[z, :(n + page - 1) // page].long()
        there = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:n]
        ids = ids.clamp(0, pages - 1)
        rows, sc = cache[ids].double().flatten(0, 1)[:n], scale[ids].double().flatten(0, 1)[:n]
        k = torch.cat([rows[:, :dc] * sc[:, :1], rows[:, dc:] * sc[:, 1:]], -1)
        k[~there] = 0.0
        place = torch.arange(n - m, n)
        q, r = q_latent[z, :, :m].double(), q_rope[z, :, :m].double()
        if rope is not None:
            r = rotate(r[None], place[None], **rope)[0]
        x = torch.cat([q, r], -1)
        s = x @ k.T * sm
        seen = there[None, :].expand(m, n)
        if causal:
            seen = seen & (torch.arange(n)[None, :] <= place[:, None])
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp(), torch.zeros_like(s))
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(total == 0, torch.ones_like(total), total)
        v = k[:, :dc]
        out[z, :, :m], mean_v[z, :, :m] = w @ v, w @ v.abs()
        # weights that are far under the row's largest one, times its token's scale, are held in steps of 2^-35 of that: half a step of it for every token's int8 numbers
        mean_v[z, :, :m] += 2.0 ** 11 * 2.0 ** -36 * (w * sc[:, 0].clamp(min=LEAST_SCALE)).amax(-1, keepdim=True) * (rows[:, :dc].abs() * there[:, None]).sum(0)
        size[z, :, :m] = (x.abs() @ k.abs().T * abs(sm) * seen).amax(-1, keepdim=True)
        step[z, :, :m] = (k.abs().sum(-1) * abs(sm) * seen).amax(-1, keepdim=True) * (x.abs().amax(-1, keepdim=True) / 32512.0 / 2.0)
        lse[z, :, :m] = torch.where(seen.any(-1), ((top + total.log()) / math.log(2.0))[..., 0], torch.full((), -math.inf, dtype=torch.float64))
    return out, lse, mean_v, size, step


def expanded(q_nope, q_rope, k_nope, k_rope, v, causal, sm, nq=None, nk=None):
    """Returns the output, lse (base 2), the mean of |v| and the largest sum of |q k| as above."""
    Z, H, N, _ = q_nope.shape
    Nk = v.shape[2]
    out, lse = torch.zeros((Z, H, N, v.shape[-1]), dtype=torch.float64), torch.full((Z, H, N), -math.inf, dtype=torch.float64)
    mean_v, size = torch.zeros_like(out), torch.zeros((Z, H, N, 1), dtype=torch.float64)
    q = torch.cat([q_nope, q_rope], -1).double()
    k = torch.cat([k_nope, k_rope.expand(-1, H, -1, -1)], -1).double()
    for z in range(Z):
        m = N if nq is None else max(0, min(int(nq[z]), N))
        n = Nk if nk is None else max(0, min(int(nk[z]), Nk))
        if m == 0 or n == 0:
            continue
        s = q[z, :, :m] @ k[z, :, :n].transpose(-1, -2) * sm
        seen = torch.ones((m, n), dtype=torch.bool)
        if causal:
            seen = torch.arange(n)[None, :] <= torch.arange(n - m, n)[:, None]
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp(), torch.zeros_like(s))
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(total == 0, torch.ones_like(total), total)
        vz = v[z, :, :n].double()
        out[z, :, :m], mean_v[z, :, :m] = w @ vz, w @ vz.abs()
        size[z, :, :m] = (q[z, :, :m].abs() @ k[z, :, :n].abs().transpose(-1, -2) * abs(sm) * seen).amax(-1, keepdim=True)
        lse[z, :, :m] = torch.where(seen.any(-1), ((top + total.log()) / math.log(2.0))[..., 0], torch.full((), -math.inf, dtype=torch.float64))
    return out, lse, mean_v, size
