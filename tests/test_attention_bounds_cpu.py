"""The bound that holds single-token attention to its definition: the kernel's
arithmetic, emulated, passes it, and mistakes planted in the emulation do not."""
import math

import pytest

torch = pytest.importorskip("torch")

from _attention import D, beyond, definition, excess, heavy_keys, lift, turned  # noqa: E402


def rnd(*shape, seed, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def two_parts(x, parts=2):
    """fp32 x as `parts` bf16 numbers, summed."""
    hi = x.to(torch.bfloat16).float()
    return hi if parts == 1 else hi + (x - hi).to(torch.bfloat16).float()


def emulated(q, k, v, pos, theta=1e6, parts=2, keep=None):
    """One sequence in 32 bits: q [Hq, 128], k and v [n, Hkv, 128]."""
    group = q.shape[0] // k.shape[1]
    x = two_parts(turned(q, pos, theta)[0].float() if theta else q.float(), parts)
    kk, vv = k.float().repeat_interleave(group, 1), v.float().repeat_interleave(group, 1)
    a = torch.matmul(kk.transpose(0, 1), x[:, :, None])[:, :, 0] / math.sqrt(D)
    if keep is not None:
        a = a.masked_fill(~keep, -math.inf)
    p = (a - a.amax(1, keepdim=True)).exp()
    return (torch.matmul(two_parts(p, parts)[:, None], vv.transpose(0, 1))[:, 0] / p.sum(1, keepdim=True)).to(torch.bfloat16)


CASES = [(1, 1, 1), (17, 4, 2), (64, 4, 2), (129, 8, 2), (300, 16, 4), (2047, 4, 1), (9000, 2, 1)]


@pytest.mark.parametrize("n,hq,hkv", CASES)
@pytest.mark.parametrize("std", [1.0, 3.0])
def test_two_part_products_pass_and_mistakes_do_not(n, hq, hkv, std):
    q, k, v = rnd(hq, D, seed=1, std=std), rnd(n, hkv, D, seed=2), rnd(n, hkv, D, seed=3)
    truth, pos = definition(q, k, v, n - 1, 1e6), torch.arange(n)

    def over(o):
        return beyond(o, *truth)

    assert over(emulated(q, k, v, n - 1)) <= 0
    assert beyond(emulated(q, k, v, n - 1, theta=0.0), *definition(q, k, v, n - 1)) <= 0
    assert over(torch.zeros(hq, D)) > 0
    if n == 1:
        return  # one key: its value whatever the query is
    assert over(emulated(q, k, v, n - 1, theta=0.0)) > 0                       # q not rotated
    assert over(emulated(q, k, v, n - 2)) > 0                                  # rotated to the position before
    assert over(emulated(q, k, v, n - 1, keep=pos < n - max(1, n // 10))) > 0  # the last tenth missing
    if n <= 300:
        assert over(emulated(q, k, v, n - 1, parts=1)) > 0                     # no lo parts


@pytest.mark.parametrize("n", [40, 300, 2047])
def test_a_lost_key_that_carries_weight_does_not_pass(n):
    q, k, v = rnd(2, D, seed=6), rnd(n, 1, D, seed=7), rnd(n, 1, D, seed=8)
    pos, heavy = torch.arange(n), heavy_keys(n)
    lift(q, k, heavy, n - 1, 1e6)
    truth = definition(q, k, v, n - 1, 1e6)
    assert beyond(emulated(q, k, v, n - 1), *truth) <= 0
    for j in heavy[::4] + heavy[-1:]:
        assert beyond(emulated(q, k, v, n - 1, keep=pos != j), *truth) > 0, j


def test_an_empty_sequence_is_zero():
    q, k = rnd(1, 2, D, seed=4), rnd(1, 5, 1, D, seed=5)
    assert excess(torch.zeros(1, 2, D), q, k, k, [0]) <= 0
    assert excess(torch.full((1, 2, D), 1e-30), q, k, k, [0]) > 0
    assert excess(torch.full((1, 2, D), math.nan), q, k, k, [3]) > 0
