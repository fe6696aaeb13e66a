"""Attention over a paged latent cache where the line of work is so long that its units grow (tables of very many columns), and so many requests that the workgroups become fewer."""
import pytest
import torch

import int_flashattention_amd as ifa
from latent_reference import attend, make_pool
from paged_reference import make_table
from test_gpu_latent_attention import bound, freqs_of, queries

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("H,N,columns", [(16, 1, 1 << 23), (64, 1, 1 << 23), (64, 3, 1 << 23), (128, 5, (1 << 24) - 1)])
def test_tables_of_very_many_columns(H, N, columns):
    """Three sequences of some thousand keys, in tables with room for 2^29 and 2^30: units of 128 keys with one tile each, of 512 and 2048 with several."""
    g, page, lens = torch.Generator().manual_seed(columns + H), 64, [3000, 5001, 70]
    pages = sum(-(-n // page) for n in lens) + 2
    pool, small = make_pool(g, pages, page, 128, 64, 0.5), make_table(g, lens, page, pages)
    table = torch.full((3, columns), -1, **I32)
    table[:, :small.shape[1]] = small.cuda()
    q, rope = queries(g, 3, H, N, 128, 64, torch.bfloat16), dict(freqs=freqs_of(32))
    out, lse = (x.cpu() for x in ifa.attention_paged_latent_int8(q[0].cuda(), q[1].cuda(), pool[0].cuda(), pool[1].cuda(), table, torch.tensor(lens, **I32), True, 0.1,
                                                                 freqs=rope["freqs"].cuda(), return_lse=True))
    want, want_lse, mean_v, size, step = attend(*q, *pool, small, lens, True, 0.1, rope=rope)
    assert ((out.double() - want).abs() <= bound(want, mean_v, size, step, out.dtype)).all()
    assert ((lse.double() - want_lse).abs() <= (step + 2.0 ** -19 * size)[..., 0] * 1.5 + 2.0 ** -14 + 2.0 ** -22 * want_lse.abs()).all()


def test_very_many_requests():
    """6 000 000 of up to 16 keys: their units times 256 workgroups pass 32 bits.  Every one is one of 136 (eight queries, seventeen lengths), to the bit."""
    g, Z, page = torch.Generator().manual_seed(5), 6_000_000, 16
    pool = [x.cuda() for x in make_pool(g, 1, page, 128, 32, 0.5)]
    few = [x.cuda() for x in queries(g, 8, 1, 1, 128, 32, torch.float16)]
    table = torch.zeros((1, 1), **I32)

    def call(which, lens):
        return ifa.attention_paged_latent_int8(few[0][which], few[1][which], *pool, table.expand(which.shape[0], 1), lens, False, 0.1, return_lse=True)
    which, lens = torch.arange(136, device="cuda") % 8, (torch.arange(136, device="cuda") // 8).int()
    want, want_lse = call(which, lens)
    ref, ref_lse, mean_v, size, step = attend(*(x[which].cpu() for x in few), *(x.cpu() for x in pool), torch.zeros((136, 1), dtype=torch.int32), lens.tolist(), False, 0.1)
    assert ((want.cpu().double() - ref).abs() <= bound(ref, mean_v, size, step, want.dtype)).all() and torch.equal(want_lse.cpu().isinf(), ref_lse.isinf())
    pick = torch.randint(0, 136, (Z,), generator=g).cuda()
    out, lse = call(which[pick], lens[pick])
    for at in range(0, Z, 1_000_000):
        part = pick[at:at + 1_000_000]
        assert torch.equal(out[at:at + 1_000_000], want[part]) and torch.equal(lse[at:at + 1_000_000], want_lse[part])
