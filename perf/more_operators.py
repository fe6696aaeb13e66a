"""Attention whose keys and values come from one latent vector a token, and the pages of a cache, as they are measured.

Kinds of pass ("op"):
  append    new latent vectors (normalised on the way where the case says so) and rotary keys (rotated on the way) into pages of int8 rows
            with two scales a token
  absorbed  attention of new tokens over such pages, with queries that are taken into the latent space already
  expanded  attention of prompts over keys and values that are expanded for every head, the rotary key shared by the heads
  beam      a step of a search with several beams: sequences that end are freed, beams forked, room made for a token, shared pages copied first
  copy      pages copied to other places of their pools
  compact   used pages moved to the first places of their pools, tables and counts with them
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
LEAST_SCALE = 2.0 ** -100          # the scale of a row of zeros
EPS = 1e-6
# what a drawn case may cost at most: a part of the largest listed ones
MAX_FLOPS, MAX_BYTES, MAX_SCORES = 2.5e11, 1.2e9, 2.5e8


def listed():
    return [
        # one token of one request: the smallest append there is
        dict(name="append_one_token", op="append", B=1, N=1, Nk=1000, dc=512, dr=64, page=64, norm=True, rotate=True, interleaved=True, dtype="bfloat16"),
        # whole prompts into an empty cache
        dict(name="append_prompts", op="append", B=4, N=4096, Nk=4096, dc=512, dr=64, page=64, norm=True, rotate=True, interleaved=False, dtype="bfloat16"),
        # one request being generated, a share of the heads: latency
        dict(name="absorbed_one_request", op="absorbed", B=1, H=16, N=1, Nk=1024, dc=512, dr=64, page=64, rotate=True, interleaved=True, causal=False,
             ragged=False, dtype="bfloat16"),
        # a batch being generated at different lengths, a share of the heads: the stream of the cache
        dict(name="absorbed_batch_ragged", op="absorbed", B=64, H=16, N=1, Nk=8192, dc=512, dr=64, page=64, rotate=True, interleaved=False, causal=False,
             ragged=True, dtype="bfloat16"),
        # all heads on one card: bound by products
        dict(name="absorbed_all_heads", op="absorbed", B=32, H=128, N=1, Nk=4096, dc=512, dr=64, page=64, rotate=False, interleaved=False, causal=False,
             ragged=False, dtype="bfloat16"),
        # drafted tokens checked at once, a smaller latent, odd heads and lengths, small pages
        dict(name="absorbed_drafts", op="absorbed", B=5, H=20, N=4, Nk=3001, dc=256, dr=32, page=16, rotate=True, interleaved=True, causal=True, ragged=True,
             dtype="float16"),
        # a long prompt with a share of the heads
        dict(name="expanded_prompt", op="expanded", B=1, H=16, N=4096, Nk=4096, dn=128, dr=64, dv=128, causal=True, ragged=False, dtype="bfloat16"),
        # small heads, a chunk against keys from before, odd and different lengths
        dict(name="expanded_ragged", op="expanded", B=3, H=10, N=777, Nk=1555, dn=64, dr=32, dv=64, causal=True, ragged=True, dtype="float16"),
        # few short sequences: latency of the bookkeeping
        dict(name="beam_step", op="beam", B=8, Nk=500, pages=256, dc=512, dr=64, page=64),
        # many beams of a large pool
        dict(name="beam_step_large", op="beam", B=256, Nk=6000, pages=20000, dc=512, dr=64, page=64),
        # sequences copied whole, one half of the pool's pages to the other
        dict(name="copy_pages", op="copy", pages=2048, n=1000, dc=512, dr=64, page=64),
        # a pool that was in use for long
        dict(name="compact_pool", op="compact", B=48, Nk=8000, pages=12000, dc=512, dr=64, page=64),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "append", "absorbed", "absorbed", "absorbed", "absorbed", "expanded", "expanded", "beam", "copy", "compact"])
        dtype = rng.choice(["float16", "bfloat16"])
        c = dict(op=op)
        if op == "expanded":
            small = rng.random() < 0.3
            N = _log(rng, 2, 4096)
            c.update(dn=64 if small else 128, dr=32 if small else 64, dv=64 if small else 128, B=_log(rng, 1, 8), H=rng.choice([4, 10, 16, 20, 32, 64]), N=N,
                     Nk=N + rng.choice([0, 0, _log(rng, 1, 4096)]), causal=rng.random() < 0.8, ragged=rng.random() < 0.4, dtype=dtype)
            if c["B"] * c["H"] * c["N"] * c["Nk"] > MAX_SCORES:
                continue
        else:
            c.update(dc=rng.choice([128, 256, 512, 512, 512]), dr=rng.choice([32, 64, 64]), page=rng.choice([16, 32, 64, 64, 128, 256]))
        if op == "append":
            N = rng.choice([1, _log(rng, 2, 4096)])
            c.update(B=_log(rng, 1, 64), N=N, Nk=N + _log(rng, 1, 1024), norm=rng.random() < 0.6, rotate=rng.random() < 0.7, interleaved=rng.random() < 0.5,
                     dtype=dtype)
        elif op == "absorbed":
            N = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 16, 256)])
            c.update(B=_log(rng, 1, 64), H=rng.choice([1, 8, 16, 20, 32, 64, 128]), N=N, Nk=N + _log(rng, 16, 65536), rotate=rng.random() < 0.6,
                     interleaved=rng.random() < 0.5, causal=N > 1, ragged=rng.random() < 0.5, dtype=dtype)
            if c["B"] * c["H"] * N * c["Nk"] > MAX_SCORES or c["B"] * c["Nk"] > 600000:
                continue
        elif op in ("beam", "compact"):
            B, Nk = _log(rng, 2, 256), _log(rng, 16, 8192)
            need = B * (-(-Nk // c["page"]) + 2)
            c.update(B=B, Nk=Nk, pages=need + _log(rng, 1, max(2, need)))
            if c["pages"] * c["page"] > 1500000:
                continue
        elif op == "copy":
            pages = _log(rng, 8, 8192)
            c.update(pages=pages, n=max(1, int(pages * rng.uniform(0.05, 0.5))))
            if pages * c["page"] > 1000000:
                continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


# ---- inputs

def _frequencies(rot):
    """Radians per position of each pair (float64)."""
    return 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=DEV) / rot)


def _key_lengths(case):
    """Keys of each entry, the new tokens among them: from all of Nk down to a quarter of it where the batch is ragged."""
    B, N, cap = case["B"], case.get("N", 1), case["Nk"]
    if not case.get("ragged"):
        return [cap] * B
    return [max(min(N, cap), cap - (cap * 3 // 4) * i // B) for i in range(B)]


def _query_lengths(case):
    """New tokens of each entry: all of N, fewer for every other entry of a ragged batch."""
    B, N = case["B"], case["N"]
    return [N if i % 2 == 0 or not case.get("ragged") else max(1, N * 5 // 8) for i in range(B)]


def _pool(g, case, pages):
    """Pages of int8 rows (latent, then rotary key) and the two scales of each token; tokens differ in magnitude, and rotary keys are larger."""
    shape = (pages, case["page"], case["dc"] + case["dr"])
    cache = torch.empty(shape, dtype=torch.int8, device=DEV)
    step = max(1, (64 << 20) // (shape[1] * shape[2]))
    for at in range(0, pages, step):
        part = cache[at:at + step]
        part.copy_((torch.randn(part.shape, generator=g, device=DEV, dtype=torch.float16) * 31.75).round().clamp(-127, 127))
    scale = (0.7 + 0.6 * torch.rand((pages, case["page"], 2), generator=g, device=DEV)) / 31.75
    scale[..., 1] *= 2.0
    return cache, scale


def _beams(case):
    """The plan of a beam step: groups of four beams of one prompt that share all its pages but each its own last ones."""
    B, page, Nk = case["B"], case["page"], case["Nk"]
    return [max(1, Nk - (Nk // 2) * (i // 4) // max(1, B // 4)) for i in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = dict(op=op)
    if op == "expanded":
        dt, B, H, N, Nk, dn, dr, dv = DTYPES[case["dtype"]], *(case[n] for n in ("B", "H", "N", "Nk", "dn", "dr", "dv"))
        q = torch.randn((B, N, H, dn + dr), generator=g, device=DEV).mul_(1.5).to(dt).transpose(1, 2)        # as projections leave them
        kv = torch.randn((B, Nk, H, dn + dv), generator=g, device=DEV).to(dt).transpose(1, 2)
        s.update(q_nope=q[..., :dn], q_rope=q[..., dn:], k_nope=kv[..., :dn], v=kv[..., dn:], k_rope=torch.randn((B, Nk, dr), generator=g, device=DEV).to(dt)[:, None],
                 causal=case["causal"], sm=(dn + dr) ** -0.5, nq=None, nk=None)
        if case["ragged"]:
            s["nq"] = torch.tensor(_query_lengths(case), dtype=torch.int32, device=DEV)
            s["nk"] = torch.tensor(_key_lengths(case), dtype=torch.int32, device=DEV)
        return s
    page, dc, dr = case["page"], case["dc"], case["dr"]
    if op in ("append", "absorbed"):
        dt, B, N = DTYPES[case["dtype"]], case["B"], case["N"]
        lens = [max(0, case["Nk"] - N - i % 7) for i in range(B)] if op == "append" else _key_lengths(case)
        width = -(-(max(lens) + (N if op == "append" else 0)) // page)
        s["cache"], s["scale"] = _pool(g, case, B * width)
        s.update(dc=dc, freqs=_frequencies(dr) if case["rotate"] else None, interleaved=case["interleaved"],
                 table=torch.randperm(B * width, generator=g, device=DEV).to(torch.int32).reshape(B, width), lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if op == "append":
            c = torch.randn((B, N, dc), generator=g, device=DEV)
            c *= 0.2 + torch.rand((B, N, 1), generator=g, device=DEV)                    # tokens differ in magnitude before their norm
            s.update(c_new=c.to(dt), k_new=(2.0 * torch.randn((B, N, dr), generator=g, device=DEV)).to(dt),
                     weight=(1.0 + 0.3 * torch.randn((dc,), generator=g, device=DEV)).to(dt) if case["norm"] else None,
                     values=torch.empty(s["cache"].shape, dtype=dt, device=DEV))
            return s
        # absorbed queries: the latent part is a product over a head's own width, as large as what it replaces
        q = torch.randn((B, case["H"], N, dc), generator=g, device=DEV).mul_(1.5 * (64.0 / dc) ** 0.5).to(dt)
        s.update(q_latent=q, q_rope=torch.randn((B, case["H"], N, dr), generator=g, device=DEV).to(dt), causal=case["causal"], sm=192.0 ** -0.5 * 1.6,
                 nq=torch.tensor(_query_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] and N > 1 else None)
        return s
    pages = case["pages"]
    s["cache"], s["scale"] = _pool(g, case, pages)
    if op == "copy":
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        s.update(src=order[:case["n"]].contiguous(), dst=order[case["n"]:2 * case["n"]].contiguous())
        return s
    B, lens = case["B"], _beams(case) if op == "beam" else [max(1, case["Nk"] - (case["Nk"] * i) // case["B"]) for i in range(case["B"])]
    width = -(-max(lens) // page) + 1
    table, refs = [[-1] * width for _ in range(B)], [0] * pages
    free = torch.randperm(pages, generator=g, device=DEV).tolist()
    for z, n in enumerate(lens):
        leader = z - z % 4
        for i in range(-(-n // page)):
            shared = op == "beam" and z != leader and i < -(-lens[leader] // page) - 1      # a page of the prompt
            table[z][i] = table[leader][i] if shared else free.pop()
            refs[table[z][i]] += 1
    table, refs = torch.tensor(table, dtype=torch.int32), torch.tensor(refs, dtype=torch.int32)
    s.update(page=page, table0=table.to(DEV), refs0=refs.to(DEV), lens0=torch.tensor(lens, dtype=torch.int32, device=DEV))
    s.update(table=torch.empty_like(s["table0"]), refs=torch.empty_like(s["refs0"]), lens=torch.empty_like(s["lens0"]))
    if op == "beam":
        # the best beams of each group take over from others; one group in eight has ended
        ended = [z for z in range(B) if z // 4 % 8 == 7]
        live = [z for z in range(B) if z // 4 % 8 != 7]
        pick = torch.randint(0, 4, (len(live),), generator=g, device=DEV).tolist()
        s.update(ended=torch.tensor(ended, dtype=torch.int32, device=DEV), children=torch.tensor(live, dtype=torch.int32, device=DEV),
                 parents=torch.tensor([min(z - z % 4 + k, live[-1]) for z, k in zip(live, pick)], dtype=torch.int32, device=DEV),
                 fresh=torch.tensor([0 if z // 4 % 8 == 7 else 1 for z in range(B)], dtype=torch.int32, device=DEV))
    return s


# ---- plain forms: elementary operations in 32 bits, angles in 64

def _rotated(x, positions, freqs, interleaved):
    """x [Z, H, N, d] in fp32, all of d rotated by positions [Z, N]."""
    angle = positions.double()[:, None, :, None] * freqs
    c, s = angle.cos().float(), angle.sin().float()
    r = x.shape[-1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :r // 2], x[..., r // 2:])
    a2, b2 = a * c - b * s, b * c + a * s
    return torch.stack([a2, b2], -1).flatten(-2) if interleaved else torch.cat([a2, b2], -1)


def _plain_append(s):
    c, k, lens, page, dc = s["c_new"].float(), s["k_new"].float(), s["lens"].long(), s["cache"].shape[1], s["dc"]
    if s["weight"] is not None:
        c = c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].float()
    positions = lens[:, None] + torch.arange(c.shape[1], device=c.device)
    if s["freqs"] is not None:
        k = _rotated(k[:, None], positions, s["freqs"], s["interleaved"])[:, 0]
    ids, row = s["table"].long().gather(1, positions // page), positions % page
    sc = torch.stack([(x.abs().amax(-1) / 127.0).clamp(min=LEAST_SCALE) for x in (c, k)], -1)
    s["cache"][ids, row] = torch.cat([(c / sc[..., :1]).round(), (k / sc[..., 1:]).round()], -1).to(torch.int8)
    s["scale"][ids, row] = sc


def _softmax_product(scores, v):
    """Rows that see no key are zeros."""
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p / torch.where(total == 0.0, 1.0, total), v)


def _plain_absorbed(s):
    lens, dc = s["lens"].long(), s["dc"]
    Z, H, N, _ = s["q_latent"].shape
    nq = torch.full_like(lens, N) if s["nq"] is None else s["nq"].long()
    row = torch.arange(N, device=lens.device)
    position = (lens - nq)[:, None] + row
    q_rope = s["q_rope"].float()
    if s["freqs"] is not None:
        q_rope = _rotated(q_rope, position, s["freqs"], s["interleaved"])
    q = torch.cat([s["q_latent"].float(), q_rope], -1)
    table = s["table"].long()
    k = s["cache"][table].float()                                         # [Z, pages, page, dc + dr]
    sc = s["scale"][table]
    k = torch.cat([k[..., :dc] * sc[..., :1], k[..., dc:] * sc[..., 1:]], -1).flatten(1, 2)
    scores = torch.matmul(q.reshape(Z, H * N, -1) * s["sm"], k.transpose(-1, -2).contiguous()).reshape(Z, H, N, -1)
    key = torch.arange(k.shape[1], device=k.device)
    seen = key < lens[:, None, None]
    if s["causal"]:
        seen = seen & (key <= position[..., None])
    seen = seen & (row < nq[:, None])[..., None]
    scores = scores.masked_fill(~seen[:, None], -math.inf).reshape(Z, H * N, -1)
    return _softmax_product(scores, k[..., :dc].contiguous()).reshape(Z, H, N, dc).to(s["q_latent"].dtype)


def _plain_expanded(s):
    q = torch.cat([s["q_nope"], s["q_rope"]], -1).float()
    Z, H, N, _ = q.shape
    Nk = s["v"].shape[2]
    k = torch.cat([s["k_nope"], s["k_rope"].expand(-1, H, -1, -1)], -1).float()
    scores = torch.matmul(q * s["sm"], k.transpose(-1, -2).contiguous())
    nq = torch.full((Z,), N, device=q.device) if s["nq"] is None else s["nq"].long()
    nk = torch.full((Z,), Nk, device=q.device) if s["nk"] is None else s["nk"].long()
    row, key = torch.arange(N, device=q.device), torch.arange(Nk, device=q.device)
    seen = (key < nk[:, None, None]) & (row < nq[:, None])[..., None]
    if s["causal"]:
        seen = seen & (key <= ((nk - nq)[:, None] + row)[..., None])
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    return _softmax_product(scores, s["v"].float()).to(s["v"].dtype)


def _named(table, pages):
    return (table >= 0) & (table < pages)


def _plain_beam(s):
    refs, table, lens, page = s["refs"], s["table"], s["lens"], s["page"]
    pages = refs.shape[0]
    # sequences that end
    old = table[s["ended"].long()]
    refs.index_add_(0, old.clamp(0, pages - 1).flatten().long(), -_named(old, pages).flatten().to(torch.int32))
    table[s["ended"].long()] = -1
    lens[s["ended"].long()] = 0
    # beams go on from their parents, all read before any is written
    new, new_lens, old = table[s["parents"].long()], lens[s["parents"].long()], table[s["children"].long()]
    refs.index_add_(0, new.clamp(0, pages - 1).flatten().long(), _named(new, pages).flatten().to(torch.int32))
    refs.index_add_(0, old.clamp(0, pages - 1).flatten().long(), -_named(old, pages).flatten().to(torch.int32))
    table[s["children"].long()] = new
    lens[s["children"].long()] = new_lens
    # room for the new token: a copy of a last page that others hold too (the last holder keeps it), a free page where one begins
    z, width = torch.arange(table.shape[0], device=table.device), table.shape[1]
    wants, column = s["fresh"] > 0, (lens // page).long()
    here = table[z, column.clamp(max=width - 1)].long()
    inside = wants & (column < width)
    part = inside & (lens % page != 0) & _named(here, pages)
    same = (here[:, None] == here[None, :]) & part[:, None] & part[None, :]
    before = (same & (z[None, :] < z[:, None])).sum(1)
    copies = part & (refs[here.clamp(0, pages - 1)] - before > 1)
    begins = inside & ~_named(here, pages)
    takes = copies | begins
    rank = takes.cumsum(0) - 1
    free = (refs <= 0).nonzero()[:, 0]
    got = takes & (rank < free.shape[0])
    page_of = free[rank.clamp(0, max(0, free.shape[0] - 1))]
    moved = got & copies
    refs.index_add_(0, here.clamp(0, pages - 1), -moved.to(torch.int32))
    refs.index_add_(0, page_of, got.to(torch.int32))
    table[z, column.clamp(max=width - 1)] = torch.where(got, page_of, here).to(torch.int32)
    s["cache"][page_of[moved]] = s["cache"][here[moved]]
    s["scale"][page_of[moved]] = s["scale"][here[moved]]
    return torch.where(inside & (got | ~takes), s["fresh"], 0)


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    pages = refs.shape[0]
    used = refs > 0
    place = torch.arange(pages, device=refs.device)
    front = place < used.sum()
    src, dst = (used & ~front).nonzero()[:, 0], (~used & front).nonzero()[:, 0]
    s["cache"][dst] = s["cache"][src]
    s["scale"][dst] = s["scale"][src]
    moved = torch.where(used, place, -1)
    moved[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(_named(table, pages), moved[table.clamp(0, pages - 1).long()].to(torch.int32), table))
    return moved.to(torch.int32)


def run(s):
    if own:
        import int_flashattention_amd as M
    op = s["op"]
    if op == "append":
        if own:
            M.paged_latent_append(s["cache"], s["scale"], s["c_new"], s["k_new"], s["table"], s["lens"], s["freqs"], interleaved=s["interleaved"],
                                  norm_weight=s["weight"], norm_eps=EPS)
        else:
            _plain_append(s)
        # the cache as the values that it stands for
        dc = s["dc"]
        torch.mul(s["cache"][..., :dc], s["scale"][..., :1], out=s["values"][..., :dc])
        torch.mul(s["cache"][..., dc:], s["scale"][..., 1:], out=s["values"][..., dc:])
        return [s["values"], s["scale"]]
    if op == "absorbed":
        if own:
            return M.attention_paged_latent_int8(s["q_latent"], s["q_rope"], s["cache"], s["scale"], s["table"], s["lens"], s["causal"], s["sm"],
                                                 freqs=s["freqs"], interleaved=s["interleaved"], seqlens_q=s["nq"])
        return _plain_absorbed(s)
    if op == "expanded":
        if own:
            return M.attention_latent(s["q_nope"], s["q_rope"], s["k_nope"], s["k_rope"], s["v"], s["causal"], s["sm"], seqlens_q=s["nq"], seqlens_k=s["nk"])
        return _plain_expanded(s)
    pools = (s["cache"], s["scale"])
    if op == "copy":
        if own:
            M.paged_copy(pools, s["src"], s["dst"])
        else:
            s["cache"][s["dst"].long()] = s["cache"][s["src"].long()]
            s["scale"][s["dst"].long()] = s["scale"][s["src"].long()]
        return list(pools)
    # the same step each time: tables, counts and lengths as they were before it
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    s["lens"].copy_(s["lens0"])
    if op == "beam":
        if own:
            M.paged_free(s["refs"], s["table"], s["lens"], s["ended"], s["page"])
            M.paged_fork(s["refs"], s["table"], s["lens"], s["parents"], s["children"])
            granted = M.paged_reserve(pools, s["refs"], s["table"], s["lens"], s["fresh"], s["page"])
        else:
            granted = _plain_beam(s)
        return [s["table"], s["refs"], s["lens"], granted, *pools]
    moved = M.paged_compact(pools, s["refs"], s["table"]) if own else _plain_compact(s)
    return [s["table"], s["refs"], moved, *pools]


# ---- what one pass cannot do without

def work(case):
    op = case["op"]
    if op == "expanded":
        B, H, N, dn, dr, dv = (case[n] for n in ("B", "H", "N", "dn", "dr", "dv"))
        lens, nq = _key_lengths(case), _query_lengths(case)
        pairs = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for m, n in zip(nq, lens))
        return {"bytes": 2.0 * H * (sum(nq) * (dn + dr) + B * N * dv + sum(lens) * (dn + dv)) + 2.0 * dr * sum(lens), "flops": 2.0 * H * pairs * (dn + dr + dv)}
    page, row = case["page"], case["dc"] + case["dr"]
    if op == "append":
        B, N = case["B"], case["N"]
        # 16-bit rows in, int8 rows and two scales out; then the pool as 16-bit values, which is returned
        pool = B * -(-case["Nk"] // page) * page
        return {"bytes": B * N * (3.0 * row + 8.0) + pool * (3.0 * row + 8.0), "flops": B * N * 6.0 * row}
    if op == "absorbed":
        B, H, N, dc = case["B"], case["H"], case["N"], case["dc"]
        lens, nq = _key_lengths(case), _query_lengths(case)
        pairs = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for m, n in zip(nq, lens))
        return {"bytes": sum(lens) * (row + 8.0) + 2.0 * B * H * N * (row + dc), "flops": 2.0 * H * pairs * (row + dc)}
    if op == "copy":
        return {"bytes": 2.0 * case["n"] * page * (row + 8.0), "flops": 0.0}
    if op == "beam":
        width = -(-case["Nk"] // page) + 1
        # tables and counts in and out, twice over (as they were, and the step); about half of the live beams copy a page
        return {"bytes": 4.0 * (4 * case["B"] * width + 4 * case["pages"]) + case["B"] * 0.4 * 2.0 * page * (row + 8.0), "flops": 0.0}
    used = sum(-(-max(1, case["Nk"] - (case["Nk"] * i) // case["B"]) // page) for i in range(case["B"]))
    # pages behind the used ones' number are used as often as the others
    return {"bytes": 2.0 * used * (1.0 - used / case["pages"]) * page * (row + 8.0) + 16.0 * case["pages"], "flops": 0.0}


# ---- the same by definition, in 64 bits

def _turned(x, position, freqs, interleaved):
    """x [..., N, d] in float64 and positions [N]: each pair as a complex number times e^(i position f)."""
    w = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(position.double(), freqs))
    if interleaved:
        return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * w).flatten(-2)
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * w
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    op = case["op"]
    if op not in ("append", "absorbed", "expanded"):
        return None                                          # whole numbers
    s = prepare(case, seed)
    if op == "append":
        held, scale, dc, page = s["cache"].double(), s["scale"].double(), s["dc"], case["page"]
        for z, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n, n + case["N"], device=DEV)
            c, k = s["c_new"][z].double(), s["k_new"][z].double()
            if s["weight"] is not None:
                c = c * torch.rsqrt(c.pow(2).mean(-1, keepdim=True) + EPS) * s["weight"].double()
            if s["freqs"] is not None:
                k = _turned(k, at, s["freqs"], s["interleaved"])
            ids = s["table"][z].long()[at // page]
            for i, (x, cols) in enumerate(((c, slice(0, dc)), (k, slice(dc, None)))):
                step = (x.abs().amax(-1) / 127.0).clamp(min=LEAST_SCALE)
                scale[ids, at % page, i] = step
                held[ids, at % page, cols] = (x / step[:, None]).round()
        return [torch.cat([held[..., :dc] * scale[..., :1], held[..., dc:] * scale[..., 1:]], -1), scale]
    if op == "expanded":
        B, H, N, Nk = (case[n] for n in ("B", "H", "N", "Nk"))
        out = torch.zeros((B, H, N, case["dv"]), dtype=torch.float64, device=DEV)
        nq, nk = _query_lengths(case), _key_lengths(case)
        for z in range(B):
            m, n = nq[z], nk[z]
            for h in range(H):
                kr, kn, v = s["k_rope"][z, 0, :n].double(), s["k_nope"][z, h, :n].double(), s["v"][z, h, :n].double()
                for at in range(0, m, 1024):
                    rows = slice(at, min(m, at + 1024))
                    score = (s["q_nope"][z, h, rows].double() @ kn.T.contiguous() + s["q_rope"][z, h, rows].double() @ kr.T.contiguous()) * s["sm"]
                    if s["causal"]:
                        place = n - m + torch.arange(m, device=DEV)[rows]
                        score = torch.where(torch.arange(n, device=DEV)[None] > place[:, None], -math.inf, score)
                        score = torch.where((place < 0)[:, None], 0.0, score)
                        out[z, h, rows] = torch.where((place < 0)[:, None], 0.0, torch.softmax(score, -1) @ v)
                    else:
                        out[z, h, rows] = torch.softmax(score, -1) @ v
        return out
    lens, table, dc = s["lens"].tolist(), s["table"], s["dc"]
    nq = [case["N"]] * len(lens) if s["nq"] is None else s["nq"].tolist()
    out = torch.zeros(s["q_latent"].shape, dtype=torch.float64, device=DEV)
    for z, (n, m) in enumerate(zip(lens, nq)):
        ids = table[z].long()[:-(-n // case["page"])]
        row = s["cache"][ids].flatten(0, 1)[:n].double()
        sc = s["scale"][ids].flatten(0, 1)[:n].double()
        c, k = row[:, :dc] * sc[:, :1], row[:, dc:] * sc[:, 1:]
        place = torch.arange(n - m, n, device=DEV)
        q, r = s["q_latent"][z, :, :m].double(), s["q_rope"][z, :, :m].double()
        if s["freqs"] is not None:
            r = _turned(r, place, s["freqs"], s["interleaved"])
        score = ((q.flatten(0, 1) @ c.T.contiguous() + r.flatten(0, 1) @ k.T.contiguous()) * s["sm"]).unflatten(0, (case["H"], m))
        if s["causal"]:
            score = torch.where(torch.arange(n, device=DEV)[None, :] > place[:, None], -math.inf, score)
        out[z, :, :m] = (torch.softmax(score, -1).flatten(0, 1) @ c).unflatten(0, (case["H"], m))
    return out
