"""Random shapes, lengths, masks, rotations, scales and page tables of the latent cache's attention and of the expanded form against their formulas in float64."""
import random

import pytest
import torch

import test_gpu_latent_attention as A
import test_gpu_latent_expanded as E
from latent_reference import make_pool
from paged_reference import make_table
from test_gpu_latent_attention import check, freqs_of, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(120))
def test_absorbed(seed, monkeypatch):
    monkeypatch.setitem(A.WIDE, "on", seed % 2 == 1)
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dc, dr, page = r.choice((128, 256, 512)), r.choice((32, 64)), r.choice((16, 32, 64, 128, 256))
    Z, N = r.choice((1, 2, 3, 7)), r.choice((1, 1, 1, 2, 3, 8, 17))
    H = r.choice((1, 2, 5, 16, 17, 24, 32, 40, 64, 100, 128) if N < 8 else (1, 3, 8, 12))
    top = r.choice((1, 40, 65, 130, 400, 1500 // Z))
    lens = [r.randint(0, top) for _ in range(Z)]
    if r.random() < 0.2:
        lens[r.randrange(Z)] = -r.randint(0, 5)
    held = [max(0, n) for n in lens]
    pages = sum(-(-n // page) for n in held) + r.randint(1, 4)
    table = make_table(g, held, page, pages, r.randint(1, 3))
    if r.random() < 0.2:
        table[r.randrange(Z), 0] = r.choice((-1, pages, -(2 ** 31)))      # a page that is none
    pairs = r.choice([p for p in (8, 16, 24, 32) if p <= dr // 2])
    rope = None if r.random() < 0.4 else dict(freqs=freqs_of(pairs), interleaved=r.random() < 0.5, magnitude=r.choice((1.0, 1.3)))
    fresh = None if N == 1 or r.random() < 0.5 else [r.randint(-1, N + 2) for _ in range(Z)]
    check(queries(g, Z, H, N, dc, dr, r.choice((torch.float16, torch.bfloat16))), make_pool(g, pages, page, dc, dr, r.choice((0.0, 0.5, 3.0))), table, lens, r.random() < 0.6,
          r.choice((0.1, 0.07, -0.05)), fresh, rope)


@pytest.mark.parametrize("seed", range(80))
def test_expanded(seed):
    r, g = random.Random(1000 + seed), torch.Generator().manual_seed(1000 + seed)
    Z, H, N, Nk = r.choice((1, 2, 4)), r.choice((1, 2, 5)), r.choice((1, 2, 31, 64, 127, 128, 129, 200, 400)), r.choice((1, 3, 63, 64, 65, 127, 190, 300, 700))
    lens = lambda n: None if r.random() < 0.5 else [r.randint(-1, n + 3) for _ in range(Z)]  # noqa: E731
    tiles = Z * H * -(-N // 128)
    E.check(E.inputs(g, Z, H, N, Nk, r.choice(E.DIMS), r.choice((torch.float16, torch.bfloat16))), r.random() < 0.6, r.choice((0.07, 0.1, -0.05)), lens(N), lens(Nk),
            copies=1 if r.random() < 0.5 else 256 // tiles + 1)
