"""Attention calls of more workgroups than one launch can have (2^32 threads)."""
import pytest
import torch

import epure
from epure.kernels import cuda
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def filled(g, n_seq, length, page, heads, dim):
    """A cache of n_seq random contexts, its table, and the contexts [n_seq, L, heads, D]."""
    width = -(-length // page)
    cache = epure.PagedKVCache(n_seq * width, page, heads, dim, BF16, DEV)
    table = torch.randperm(n_seq * width, generator=g, device=DEV).to(torch.int32).view(n_seq, width)
    pos = torch.arange(length, device=DEV).expand(n_seq, length)
    k, v = (torch.randn(n_seq, length, heads, dim, generator=g, device=DEV) for _ in range(2))
    cache.append(k, v, pos, table)
    return cache, table, op.stands_for(k, BF16), op.stands_for(v, BF16)


def check(out, q, pos, kc, vc, D):
    """Rows [n, S, heads, D] against the oracle over their contexts."""
    want, mag, big = op.attend(q, kc, vc, pos.cpu(), D ** -0.5)
    err = (out.cpu().double() - want).abs()
    assert (err <= op.attend_tolerance(want, mag, big, BF16, D)).all()


def test_more_segments_than_one_launch_takes():
    """2^24 + 24 workgroups of one segment each: two launches."""
    g = torch.Generator(device=DEV).manual_seed(1)
    B, H, D = (1 << 21) + 3, 8, 16
    cache, table, kc, vc = filled(g, 5, 16, 16, H, D)
    of = torch.arange(B, device=DEV) % 5                # five contexts, each of many sequences
    q = torch.randn(B, 1, H, D, generator=g, device=DEV, dtype=BF16)
    pos = torch.randint(0, 16, (B, 1), generator=g, device=DEV)
    out = cache.attend(q, pos, table[of])
    most = (1 << 24) - 1                                # workgroups of the first launch
    at = torch.tensor([0, 1, B // 3, most // H - 1, most // H, most // H + 1, B - 2, B - 1], device=DEV)
    check(out[at], q[at], pos[at], kc[of[at].cpu()], vc[of[at].cpu()], D)
    # sequences of one context and position, of equal queries, are equal all over
    q[:], pos[:] = q[0], 9
    out = cache.attend(q, pos, table[of])
    for i in range(5):
        same = out[i::5]
        assert torch.equal(same, same[:1].expand_as(same))


def test_more_joined_rows_than_one_launch_takes():
    """2^25 + 160 output rows, whose work is shared and whose pieces are joined
    by a workgroup of 128 threads each."""
    g = torch.Generator(device=DEV).manual_seed(2)
    B, S, G, D, L = 2, (1 << 20) + 5, 16, 16, 1120
    cache, table, kc, vc = filled(g, B, L, 16, 1, D)
    q = torch.randn(B, S, G, D, generator=g, device=DEV, dtype=BF16)
    pos = torch.randint(0, L, (B, S), generator=g, device=DEV)
    assert B * S * G > 1 << 25
    out = cache.attend(q, pos, table)
    at = torch.cat((torch.arange(8), torch.randint(0, S, (48,)), torch.arange(S - 16, S))).to(DEV)
    check(out[:, at], q[:, at], pos[:, at], kc, vc, D)
    # every row again, in calls that share their work otherwise: the same to
    # the output's rounding and what 2^-14 of a mean of values below 6 can be off
    part = S // 16 + 1
    for s in range(0, S, part):
        again = cache.attend(q[:, s:s + part], pos[:, s:s + part], table).float()
        assert ((out[:, s:s + part].float() - again).abs() <= 2.0 ** -7 * again.abs() + 6 * 2.0 ** -13).all()
