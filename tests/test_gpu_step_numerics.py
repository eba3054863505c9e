"""GPU: how exact the paged decode attention's weights are, on inputs whose scores carry no rounding
that could hide them.

A query with a single non-zero component makes every product but one of a score zero: the sum is
exact, and the score x (log2 units, at most 8 here) is off only by its scale factors' roundings:
constant, product with the softmax scale, the query's power of two, the K scale, the last product --
5 * 2^-24 * 8 < 2^-18; the subtraction of the running maximum adds 2^-24 * 16, the exponential
2^-22, so a weight is off by less than 2^-18 relative, and o by 2^-17 a, a = sum w |v| / sum w, as
the weights stand above and below the division.  The weights are carried in two float16 halves
(2^-22 relative, 2^-25 of the largest below that), n of them are summed above and below (2 n 2^-24),
and the codes' bias adds 48 * 2^-24 max|v| (18 roundings of 2.1 max|v|).
"""

import math

import numpy as np
import pytest
import torch

from oracle import step as ostep

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 (B200) device")
    from kvboost_b200 import ops
    ops.read_status(torch.device("cuda"))
    yield
    assert ops.read_status(torch.device("cuda")) == 0


def _half_step(x, dtype):
    """Half the distance between neighbours of ``dtype`` at |x|."""
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).tiny
    return 2.0 ** np.floor(np.log2(np.maximum(np.abs(x), tiny))) * eps / 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,group", [(64, 4), (96, 4), (128, 4), (64, 12), (128, 12)])
def test_int8_weights_keep_their_bits(dtype, D, group):
    """Over an int8 pool the result is the exact one rounded once: a float16 weight (2^-12 off on
    average) would move several percent of these outputs past a rounding border."""
    from kvboost_b200.paged_decode import paged_decode_attention
    B, H, n = 8, 2, 40
    g = torch.Generator().manual_seed(D + group)
    tables = torch.randperm(B * 3, generator=g).view(B, 3).to(torch.int32)
    pool = torch.randint(-127, 128, (B * 3, 2, H, 16, D), generator=g).to(torch.int8)
    ks = (0.5 + torch.rand(B * 3, H, 16, generator=g)).div(64).to(torch.float16)
    vs = (0.5 + torch.rand(B * 3, H, D, generator=g)).div(64).to(torch.float16)
    q = torch.zeros(B, H * group, 1, D)
    at = torch.randint(0, D, (B, H * group, 1, 1), generator=g)
    q.scatter_(3, at, torch.randint(-3, 4, at.shape, generator=g).float())
    q = q.to(dtype)
    scale = 0.5                               # |score| <= 0.5 * 3 * 127 * 1.5 / 64 = 4.5, 6.5 in log2
    lens = [n] * B
    o, _ = paged_decode_attention(q.cuda(), pool.cuda(), tables.cuda(),
                                  torch.tensor(lens, dtype=torch.int32, device=DEV), ks.cuda(), vs.cuda(),
                                  softmax_scale=scale)
    want, _, a, _, vmax, _, _ = ostep.decode_attention(q[:, :, 0].float().numpy(), pool.numpy(), tables.numpy(), lens,
                                                       scale, ks.float().numpy(), vs.float().numpy())
    got = o[:, :, 0].double().cpu().numpy()
    off = (2.0 ** -17 + 2.0 ** -22 + 2 * n * 2.0 ** -24) * a + (48 * 2.0 ** -24 + n * 2.0 ** -25) * vmax[..., None]
    bound = np.maximum(_half_step(want, dtype), _half_step(got, dtype)) + off
    bad = np.abs(got - want) > bound
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:4], (np.abs(got - want) / bound).max())


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True),
                                        (torch.bfloat16, True)])
@pytest.mark.parametrize("B,n,every", [(64, 2000, 160), (256, 8000, 1000)])
def test_small_weights_are_kept(dtype, int8, B, n, every):
    """Tokens of weight 2^-25.05, each below half of float16's smallest step, with large V beside a few
    tokens of weight 1 and V 0: the result is their sum alone.  Scores as above (|x| 25.05: 2^-16 of
    a, the exponential and subtraction included); in float16 halves 2^-36 of the largest weight may
    be lost per token."""
    from kvboost_b200.paged_decode import paged_decode_attention
    D, nb = 64, n // 16
    tail = torch.arange(n) % every != 0
    pool = torch.zeros(nb, 2, 1, 16, D)
    k = torch.where(tail, -127.0 if int8 else -25.046875, 0.0).view(nb, 16)
    v = torch.where(tail, 127.0 if int8 else 60000.0, 0.0).view(nb, 16)
    pool[:, 0, 0, :, 5] = k
    pool[:, 1, 0] = v[..., None]
    ks = vs = None
    if int8:
        pool = pool.to(torch.int8)
        ks = torch.full((nb, 1, 16), 25.05 / 127).to(torch.float16)
        vs = torch.full((nb, 1, D), 400.0).to(torch.float16)
    else:
        pool = pool.to(dtype)
    q = torch.zeros(B, 1, 1, D)
    q[..., 5] = 1.0
    q = q.to(dtype)
    tables = torch.arange(nb, dtype=torch.int32).repeat(B, 1)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    f = lambda t: None if t is None else t.float().numpy()  # noqa: E731
    o, lse = paged_decode_attention(q.cuda(), pool.cuda(), tables.cuda(),
                                    torch.full((B,), n, dtype=torch.int32, device=DEV), c(ks), c(vs),
                                    softmax_scale=math.log(2.0))
    want, wl, a, _, vmax, _, _ = ostep.decode_attention(
        f(q[:1, :, 0]), pool.numpy() if int8 else f(pool), tables[:1].numpy(), [n], math.log(2.0), f(ks), f(vs))
    got = o[:, :, 0].double().cpu().numpy()
    off = (2.0 ** -16 + 2 * n * 2.0 ** -24) * a + ((48 * 2.0 ** -24 if int8 else 0) + n * 2.0 ** -36) * vmax[..., None]
    bound = np.maximum(_half_step(want, dtype), _half_step(got, dtype)) + off
    assert (np.abs(got - want) <= bound).all(), (got.min(), got.max(), want.min(), want.max())
    gl = lse[:, :, 0].double().cpu().numpy()
    assert np.abs(gl - wl).max() <= 2.0 ** -18 + 2 * n * 2.0 ** -24
