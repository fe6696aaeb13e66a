"""The operators of a serving step over a paged int8 cache, as they are measured: rotary positions, the append of new keys
and values to the pages, and the attention that reads them.

Three kinds of pass ("op"):
  rotary   the rotation of a whole [Z, H, N, d] tensor by its positions, or its transpose (what a gradient goes through)
  append   new keys (rotated on the way) and values into pages of int8 rows that share one scale per page and head
  attend   attention of new tokens (queries rotated on the way where the case says so) over such a cache
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
LEAST_SCALE = 2.0 ** -100          # the scale of a page that holds nothing but zeros
# what a drawn case may cost at most: a part of the largest listed ones
MAX_FLOPS, MAX_BYTES, MAX_SCORES = 1.2e11, 1.0e9, 2.5e8


def listed():
    return [
        # the queries of one generated token: nothing but latency
        dict(name="rotary_one_token", op="rotary", B=1, H=32, N=1, D=128, rot=128, interleaved=False, inverse=False, scaling="none",
             dtype="float16"),
        # the gradient of a batch of prompts on its way back through the rotation, frequencies stretched by parts for long contexts
        dict(name="rotary_prompt_gradient", op="rotary", B=4, H=32, N=4096, D=128, rot=128, interleaved=False, inverse=True,
             scaling="parts", dtype="bfloat16"),
        # half of the head rotated in adjacent pairs, ragged length, positions scaled linearly
        dict(name="rotary_partial_ragged", op="rotary", B=2, H=16, N=3333, D=64, rot=32, interleaved=True, inverse=False,
             scaling="linear", dtype="float16"),
        # one token of one request: the smallest append there is, into a page that holds others already
        dict(name="append_one_token", op="append", B=1, Hkv=8, N=1, Nk=1000, D=128, page=64, rot=128, interleaved=False,
             scaling="none", dtype="float16"),
        # a batch of requests at different lengths, one token each, small pages
        dict(name="append_batch_step", op="append", B=64, Hkv=8, N=1, Nk=64, D=128, page=16, rot=64, interleaved=True, scaling="none",
             dtype="bfloat16"),
        # whole prompts into an empty cache
        dict(name="append_prompts", op="append", B=4, Hkv=8, N=4096, Nk=4096, D=128, page=64, rot=128, interleaved=False,
             scaling="parts", dtype="bfloat16"),
        # one request being generated against a short cache: latency again
        dict(name="attend_one_request", op="attend", B=1, H=32, Hkv=8, N=1, Nk=1024, D=128, page=64, rot=128, interleaved=False,
             scaling="none", causal=False, ragged=False, dtype="float16"),
        # a batch being generated at different lengths, grouped heads, small pages
        dict(name="attend_batch_ragged", op="attend", B=16, H=32, Hkv=8, N=1, Nk=8192, D=128, page=16, rot=128, interleaved=False,
             scaling="none", causal=False, ragged=True, dtype="bfloat16"),
        # ungrouped heads, full caches: the stream of K and V at its largest
        dict(name="attend_ungrouped", op="attend", B=32, H=32, Hkv=32, N=1, Nk=4096, D=128, page=64, rot=0, interleaved=False,
             scaling="none", causal=False, ragged=False, dtype="float16"),
        # one very long request: few heads share the card along the keys
        dict(name="attend_long_context", op="attend", B=1, H=32, Hkv=8, N=1, Nk=131072, D=128, page=128, rot=128, interleaved=False,
             scaling="parts", causal=False, ragged=False, dtype="bfloat16"),
        # drafted tokens checked at once, head_dim 64, odd lengths
        dict(name="attend_drafts", op="attend", B=4, H=16, Hkv=16, N=5, Nk=3001, D=64, page=32, rot=32, interleaved=True,
             scaling="none", causal=True, ragged=True, dtype="float16"),
        # a chunk of long prompts against the cache that holds what came before, of different lengths in the batch
        dict(name="attend_chunk", op="attend", B=2, H=32, Hkv=8, N=512, Nk=7680, D=128, page=64, rot=128, interleaved=False,
             scaling="none", causal=True, ragged=True, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["rotary", "append", "append", "attend", "attend", "attend"])
        D = rng.choice([64, 128, 128, 256])
        c = dict(op=op, D=D, rot=rng.choice([D // 2, D, D]), interleaved=rng.random() < 0.4, dtype=rng.choice(["float16", "bfloat16"]),
                 scaling=rng.choice(["none", "none", "linear", "parts"]))
        if op == "rotary":
            c.update(B=_log(rng, 1, 8), H=rng.choice([8, 12, 16, 32]), N=_log(rng, 1, 8192), inverse=rng.random() < 0.4)
        else:
            Hkv, page = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([16, 32, 64, 64, 128, 256])
            c.update(Hkv=Hkv, page=page)
            if op == "append":
                N = rng.choice([1, _log(rng, 2, 4096)])
                c.update(B=_log(rng, 1, 64), N=N, Nk=N + _log(rng, 1, 1024))
            else:
                N = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 16, 2048)])
                c.update(B=_log(rng, 1, 32), H=Hkv * rng.choice([1, 2, 4, 5, 8]), N=N, Nk=N + _log(rng, 64, 32768), causal=N > 1,
                         ragged=rng.random() < 0.5, rot=rng.choice([0, c["rot"]]))
                if c["H"] > 64 or c["B"] * c["H"] * N * c["Nk"] > MAX_SCORES:
                    continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


# ---- inputs

def _frequencies(rot, scaling):
    """Radians per position of each pair (float64) and the factor of the rotated values."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    if scaling == "linear":                                  # positions four times as dense
        return 10000.0 ** (-2.0 * i / rot) / 4.0, 1.0
    if scaling == "parts":                                   # slow pairs eight times as dense, fast ones as they are
        f = 500000.0 ** (-2.0 * i / rot)
        turns = 4096.0 * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / 8.0), 0.1 * math.log(8.0) + 1.0
    return 10000.0 ** (-2.0 * i / rot), 1.0


def _key_lengths(case):
    """Keys of each entry, the new tokens among them: from all of Nk down to a quarter of it where the batch is ragged."""
    B, N, cap = case["B"], case["N"], case["Nk"]
    if not case.get("ragged"):
        return [cap] * B
    return [max(min(N, cap), cap - (cap * 3 // 4) * i // B) for i in range(B)]


def _query_lengths(case):
    """New tokens of each entry: all of N, fewer for every other entry of a ragged batch."""
    B, N = case["B"], case["N"]
    return [N if i % 2 == 0 or not case.get("ragged") else max(1, N * 5 // 8) for i in range(B)]


def _pages(g, case, lens):
    """A pool of pages (int8 rows ~ N(0, 1) in the page's scale, K and V side by side), its scales, and the pages of each entry
    in shuffled order.  Pages differ in magnitude, as tokens do."""
    B, Hkv, D, page = (case[n] for n in ("B", "Hkv", "D", "page"))
    width = -(-max(lens) // page)
    n = B * width
    kv = (torch.randn((n, 2, Hkv, page, D), generator=g, device=DEV, dtype=torch.float16) * 31.75).round().clamp(-127, 127).to(torch.int8)
    scale = (0.7 + 0.6 * torch.rand((n, 2, Hkv), generator=g, device=DEV)) / 31.75
    table = torch.randperm(n, generator=g, device=DEV).to(torch.int32).reshape(B, width)
    return kv, scale, table


def prepare(case, seed):
    dt, D, B, N = DTYPES[case["dtype"]], case["D"], case["B"], case["N"]
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(op=case["op"], interleaved=case["interleaved"], freqs=None, magnitude=1.0)
    if case["rot"]:
        s["freqs"], s["magnitude"] = _frequencies(case["rot"], case["scaling"])
    if case["op"] == "rotary":
        s.update(x=torch.randn((B, case["H"], N, D), generator=g, device=DEV).to(dt), inverse=case["inverse"],
                 positions=torch.randint(0, 100000, (B,), generator=g, device=DEV, dtype=torch.int32))
        return s
    if case["op"] == "append":
        lens = [max(0, case["Nk"] - N - i % 7) for i in range(B)]
        kv, scale, table = _pages(g, case, [n + N for n in lens])
        k_new = torch.randn((B, case["Hkv"], N, D), generator=g, device=DEV)
        k_new[..., 5::64] *= 2.0                             # projected keys have channels that are larger than the others
        v_new = torch.randn((B, case["Hkv"], N, D), generator=g, device=DEV)
        s.update(kv=kv, scale=scale, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), k_new=k_new.to(dt),
                 v_new=v_new.to(dt), values=torch.empty(kv.shape, dtype=dt, device=DEV))
        return s
    lens = _key_lengths(case)
    kv, scale, table = _pages(g, case, lens)
    q = (2.0 * torch.randn((B, case["H"], N, D), generator=g, device=DEV)).to(dt)
    s.update(kv=kv, scale=scale, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), q=q, causal=case["causal"], sm=D ** -0.5,
             nq=torch.tensor(_query_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] and N > 1 else None)
    return s


# ---- plain forms: elementary operations in 32 bits, angles in 64

def _rotated(x, positions, freqs, magnitude, interleaved, inverse):
    """x [Z, H, N, d] in fp32, positions [Z, N]."""
    angle = positions.double()[:, None, :, None] * freqs
    c, s = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    if inverse:
        s = -s
    r = 2 * freqs.numel()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    a2, b2 = a * c - b * s, b * c + a * s
    y = torch.stack([a2, b2], -1).flatten(-2) if interleaved else torch.cat([a2, b2], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotary(s):
    x = s["x"]
    positions = s["positions"][:, None] + torch.arange(x.shape[2], device=x.device)
    return _rotated(x.float(), positions, s["freqs"], s["magnitude"], s["interleaved"], s["inverse"]).to(x.dtype)


def _plain_fill(cache, scale, x, table, lens):
    """The new rows x [Z, H, N, d] (fp32) into cache [pages, H, page, d] at positions lens + 0 .. N - 1, in place."""
    Z, H, N, d = x.shape
    page = cache.shape[2]
    lens = lens.long()
    first = lens // page
    touched = (lens + N - 1) // page - first + 1
    t = torch.arange((N + page - 2) // page + 1, device=x.device)
    t = torch.where(t < touched[:, None], t, 0)                           # (pages that an entry does not reach: its first one again)
    start = (first[:, None] + t) * page                                   # position of a page's first row
    ids = table.long().gather(1, first[:, None] + t)                      # [Z, T]
    pos = start[..., None] + torch.arange(page, device=x.device)          # [Z, T, page]
    j = pos - lens[:, None, None]
    new = (j >= 0) & (j < N)
    rows = x.transpose(1, 2)[torch.arange(Z, device=x.device)[:, None, None], j.clamp(0, N - 1)]       # [Z, T, page, H, d]
    rows, new = rows.transpose(2, 3), new[:, :, None, :, None]
    held = (start < lens[:, None])[..., None]                             # pages with rows from before
    amax = torch.where(new, rows.abs(), 0.0).amax((-1, -2))               # [Z, T, H]
    old = torch.where(held, scale[ids], 0.0)
    s = torch.maximum(torch.clamp(amax / 127.0, min=LEAST_SCALE), old)
    was = cache[ids]                                                      # [Z, T, H, page, d]
    kept = torch.where((pos < lens[:, None, None])[:, :, None, :, None], (was.float() * (old / s)[..., None, None]).round().to(torch.int8), was)
    cache[ids] = torch.where(new, (rows / s[..., None, None]).round().clamp(-127, 127).to(torch.int8), kept)
    scale[ids] = s


def _plain_append(s):
    kv, scale, lens = s["kv"], s["scale"], s["lens"]
    k, v = s["k_new"].float(), s["v_new"].float()
    if s["freqs"] is not None:
        k = _rotated(k, lens[:, None] + torch.arange(k.shape[2], device=k.device), s["freqs"], s["magnitude"], s["interleaved"], False)
    _plain_fill(kv[:, 0], scale[:, 0], k, s["table"], lens)
    _plain_fill(kv[:, 1], scale[:, 1], v, s["table"], lens)


def _plain_attend(s):
    q, lens = s["q"].float(), s["lens"].long()
    Z, H, N, d = q.shape
    nq = torch.full_like(lens, N) if s["nq"] is None else s["nq"].long()
    row = torch.arange(N, device=q.device)
    position = (lens - nq)[:, None] + row                                 # [Z, N]
    if s["freqs"] is not None:
        q = _rotated(q, position, s["freqs"], s["magnitude"], s["interleaved"], False)
    table = s["table"].long()
    rows = (s["kv"][table].float() * s["scale"][table][..., None, None]).permute(2, 0, 3, 1, 4, 5)      # [2, Z, Hkv, pages, page, d]
    Hkv = rows.shape[2]
    k, v = rows.reshape(2, Z, Hkv, -1, d)
    scores = torch.matmul(q.reshape(Z, Hkv, H // Hkv * N, d) * s["sm"], k.transpose(-1, -2).contiguous()).reshape(Z, H, N, -1)
    key = torch.arange(k.shape[2], device=q.device)
    seen = key < lens[:, None, None]
    if s["causal"]:
        seen = seen & (key <= position[..., None])
    seen = seen & (row < nq[:, None])[..., None]                          # [Z, N, keys]
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / torch.where(total == 0.0, 1.0, total)).reshape(Z, Hkv, H // Hkv * N, -1), v)
    return o.reshape(Z, H, N, d).to(s["q"].dtype)


def run(s):
    if own:
        import int_flashattention_amd as M
        turn = dict(interleaved=s["interleaved"], magnitude=s["magnitude"])
    if s["op"] == "rotary":
        return M.rotary(s["x"], s["positions"], s["freqs"], inverse=s["inverse"], **turn) if own else _plain_rotary(s)
    if s["op"] == "append":
        if own:
            kv, scale = s["kv"], s["scale"]
            M.paged_kvcache_append(kv[:, 0], scale[:, 0], kv[:, 1], scale[:, 1], s["k_new"], s["v_new"], s["table"], s["lens"], s["freqs"],
                                   **turn)
        else:
            _plain_append(s)
        # the cache as the values that it stands for
        return [torch.mul(s["kv"], s["scale"][..., None, None], out=s["values"]), s["scale"]]
    if own:
        kv, scale = s["kv"], s["scale"]
        return M.attention_paged_int8(s["q"], kv[:, 0], kv[:, 1], scale[:, 0], scale[:, 1], s["table"], s["lens"], s["causal"], s["sm"],
                                      freqs=s["freqs"], seqlens_q=s["nq"], **turn)
    return _plain_attend(s)


# ---- what one pass cannot do without

def work(case):
    B, N, D = case["B"], case["N"], case["D"]
    if case["op"] == "rotary":
        n = B * case["H"] * N
        return {"bytes": 4.0 * n * D + 4.0 * case["rot"] + 4.0 * B, "flops": 3.0 * n * case["rot"]}
    Hkv, page = case["Hkv"], case["page"]
    if case["op"] == "append":
        # 16-bit rows in, int8 rows and the scales of the reached pages out; then the pool as 16-bit values, which is returned
        n, pool = B * Hkv * N, B * -(-case["Nk"] // page) * 2 * Hkv
        return {"bytes": 6.0 * n * D + 3.0 * pool * page * D + 4.0 * pool, "flops": 3.0 * n * case["rot"] + 4.0 * n * D}
    H, lens, nq = case["H"], _key_lengths(case), _query_lengths(case)
    pairs = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for m, n in zip(nq, lens))
    keys, pages = sum(lens), sum(-(-n // page) for n in lens)
    return {"bytes": Hkv * (2.0 * D * keys + 8.0 * pages) + 4.0 * pages + 4.0 * D * H * B * N, "flops": 4.0 * H * D * pairs}


# ---- the same by definition, in 64 bits

def _turned(x, position, s, sign):
    """x [..., N, d] in float64 and positions [N]: each pair as a complex number times magnitude e^(i sign position f)."""
    r = 2 * s["freqs"].numel()
    w = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEV), sign * torch.outer(position.double(), s["freqs"]))
    y = x.clone()
    if s["interleaved"]:
        y[..., :r] = torch.view_as_real(torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) * w).flatten(-2)
    else:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * w
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rotary":
        x, first = s["x"].double(), s["positions"].tolist()
        steps = torch.arange(x.shape[2], device=DEV)
        return torch.stack([_turned(x[z], first[z] + steps, s, -1.0 if s["inverse"] else 1.0) for z in range(len(first))])
    lens, table, kv = s["lens"].tolist(), s["table"].tolist(), s["kv"]
    if s["op"] == "append":
        page, N = case["page"], case["N"]
        held, scale = kv.double(), s["scale"].double()
        for z, n in enumerate(lens):
            k, v = s["k_new"][z].double(), s["v_new"][z].double()
            if s["freqs"] is not None:
                k = _turned(k, n + torch.arange(N, device=DEV), s, 1.0)
            at = n
            while at < n + N:                                 # page by page
                p, r = table[z][at // page], at % page
                m = min(page - r, n + N - at)
                new = torch.stack([k[:, at - n:at - n + m], v[:, at - n:at - n + m]])                # [2, Hkv, m, d]
                least = (new.abs().amax((-1, -2)) / 127.0).clamp(min=LEAST_SCALE)
                to = torch.maximum(least, scale[p]) if r else least
                held[p, :, :, :r] = (held[p, :, :, :r] * (scale[p] / to)[..., None, None]).round()
                held[p, :, :, r:r + m] = (new / to[..., None, None]).round().clamp(-127, 127)
                scale[p] = to
                at += m
        return [held * scale[..., None, None], scale]
    N, causal = case["N"], s["causal"]
    nq = [N] * len(lens) if s["nq"] is None else s["nq"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["H"] // case["Hkv"]
    for z, (n, m) in enumerate(zip(lens, nq)):
        ids = torch.tensor(table[z][:-(-n // case["page"])], device=DEV)
        place = torch.arange(n - m, n, device=DEV)
        q = s["q"][z, :, :m].double()
        if s["freqs"] is not None:
            q = _turned(q, place, s, 1.0)
        for h in range(case["Hkv"]):
            k, v = ((kv[ids, i, h].double() * s["scale"][ids, i, h].double()[:, None, None]).flatten(0, 1)[:n].contiguous() for i in (0, 1))
            mine = slice(h * group, (h + 1) * group)
            score = (q[mine].flatten(0, 1) @ k.T.contiguous()).unflatten(0, (group, m)) * s["sm"]
            if causal:
                score = torch.where(torch.arange(n, device=DEV)[None, :] > place[:, None], -math.inf, score)
            out[z, mine, :m] = (torch.softmax(score, -1).flatten(0, 1) @ v).unflatten(0, (group, m))
    return out
