"""Single-token attention against a cache on the GPU, against its definition in
64 bits.

Tolerance: the output is one bf16 rounding (2^-8 relative at most).  The
weights are rounded to bf16 before the second product, which moves the output
by at most 2^-8 max|v|.  With rope, q is rounded to bf16 after the rotation: a
score moves by at most 2^-8 sum|q k| / sqrt(128), and the output by at most
twice that times max|v|; `qk` is the largest of those sums in the case at hand.
Sums are fp32 and add far less; one part in a hundred more is allowed."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import _attention  # noqa: E402

from ennx_b200 import ops  # noqa: E402

D = 128


def rnd(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def turn(x, pos, theta):
    inv = theta ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    c, s = (pos * inv).cos(), (pos * inv).sin()
    x1, x2 = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def check(got, q, kc, vc, lengths, theta=0.0):
    """got against the definition over the caches as they are now."""
    for b, n in enumerate(lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        group = q.shape[1] // kc.shape[2]
        qq = turn(q[b], n - 1, theta) if theta else q[b].double()
        kk = kc[b, :n].double().repeat_interleave(group, 1)
        vv = vc[b, :n].double().repeat_interleave(group, 1)
        a = torch.einsum("hd,jhd->hj", qq, kk) / math.sqrt(D)
        ref = torch.einsum("hj,jhd->hd", a.softmax(-1), vv)
        vmax = float(vv.abs().max())
        bound = 2.0 ** -8 * (ref.abs() + vmax)
        if theta:
            qk = torch.einsum("hd,jhd->hj", qq.abs(), kk.abs()).max() / math.sqrt(D)
            bound = bound + 2 * 2.0 ** -8 * float(qk) * vmax
        err = (got[b].double() - ref).abs() - 1.01 * bound
        assert err.max() <= 0, (b, n, float(err.max()))


# a room that fits a cluster of blocks per head, 2048 tokens each, is not split over the device
CASES = [
    (16, [1], 1, 1), (16, [16], 4, 1), (64, [17, 0, 63, 64], 4, 2), (300, [65, 299, 300], 16, 4),
    (1024, [1024, 1000, 1, 0, 129], 8, 2), (1025, [1025], 4, 4), (2048, [1, 0, 2048, 64, 65, 2047, 0], 16, 4),
    (5000, [4999, 3, 0, 0, 127, 128, 129], 16, 1), (40000, [40000], 4, 2), (3000, [2999], 17, 1), (1500, [1400, 20], 64, 2),
    (1100, [0, 0, 0], 4, 2), (2000, [11] * 200, 2, 1),
    (200, [200, 77, 0], 24, 2), (500, [500, 31, 256, 257], 9, 3), (9000, [8999, 1, 4097], 32, 2), (1300, [1300, 3] * 25, 16, 2),
    (600, [7, 600, 0, 33, 600, 1] * 20, 8, 4), (9000, [8999, 5, 300, 0, 4097, 9000] * 4, 16, 4), (300, [1, 300] * 70, 4, 4),
    (20000, [19999, 3, 0, 0, 127, 128, 129], 16, 1), (17000, [1, 0, 16999, 64, 65, 2047, 0], 16, 4), (16385, [16385], 4, 4),
    (17000, [2999], 17, 1), (17000, [1400, 20], 64, 2), (17000, [0, 0, 0], 4, 2), (2100, [11, 2100] * 100, 2, 1),
]


@pytest.mark.parametrize("room,lengths,hq,hkv", CASES)
@pytest.mark.parametrize("heads_first", [False, True])
def test_matches_definition(room, lengths, hq, hkv, heads_first):
    batch = len(lengths)
    shape = (batch, hkv, room, D) if heads_first else (batch, room, hkv, D)
    kc, vc = rnd(*shape, seed=1), rnd(*shape, seed=2)
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    for b, n in enumerate(lengths):  # what a fresh cache may hold
        kc[b, n:], vc[b, n:] = math.nan, math.inf
    k0, v0 = kc.clone(), vc.clone()
    q = rnd(batch, hq, D, seed=3)
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), rope_theta=0.0)
    check(o, q, kc, vc, lengths)
    assert torch.equal(kc.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), v0.view(torch.int16))


@pytest.mark.parametrize("room,lengths,hq,hkv", [c for c in CASES if sum(c[1])])
def test_appends_the_new_token(room, lengths, hq, hkv):
    batch, theta = len(lengths), 1e6
    kc, vc = rnd(batch, room, hkv, D, seed=4), rnd(batch, room, hkv, D, seed=5)
    for b, n in enumerate(lengths):
        kc[b, max(0, n - 1):], vc[b, max(0, n - 1):] = math.nan, math.inf
    k0, v0 = kc.clone(), vc.clone()
    fused = rnd(batch, (hq + 2 * hkv) * D, seed=6)
    q = fused[:, :hq * D].unflatten(1, (hq, D))
    k = fused[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D))
    v = fused[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
    before = fused.clone()
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), k=k, v=v, rope_theta=theta)
    for b, n in enumerate(lengths):
        if n:
            ref = turn(k[b], n - 1, theta)
            assert ((kc[b, n - 1].double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 1e-5).all()
            assert torch.equal(vc[b, n - 1], v[b])
            k0[b, n - 1], v0[b, n - 1] = kc[b, n - 1], vc[b, n - 1]
    check(o, q, kc, vc, lengths, theta)
    assert torch.equal(fused, before)
    assert torch.equal(kc.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), v0.view(torch.int16))


def test_new_token_without_rope_and_out_with_a_stride():
    kc, vc = rnd(2, 1200, 2, D, seed=7), rnd(2, 1200, 2, D, seed=8)
    q, k, v = rnd(2, 4, D, seed=9), rnd(2, 2, D, seed=10), rnd(2, 2, D, seed=11)
    wide = torch.full((2, 4 * D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.gqa_attention_decode(q, kc, vc, i32([700, 1]), k=k, v=v, rope_theta=0.0, out=wide[:, :4 * D].unflatten(1, (4, D)))
    assert torch.equal(kc[0, 699], k[0]) and torch.equal(kc[1, 0], k[1]) and torch.equal(vc[0, 699], v[0])
    check(wide[:, :4 * D].unflatten(1, (4, D)), q, kc, vc, [700, 1])
    assert (wide[:, 4 * D:] == 5.0).all()


@pytest.mark.parametrize("room,hq", [(200, 4), (300, 4), (3000, 4), (3000, 40), (17000, 4), (17000, 40)])
def test_out_may_be_the_queries(room, hq):
    kc, vc, q = rnd(3, room, 2, D, seed=50), rnd(3, room, 2, D, seed=51), rnd(3, hq, D, seed=52)
    want, ln = q.clone(), i32([room, 0, 77])
    ref = ops.gqa_attention_decode(want, kc, vc, ln)
    assert torch.equal(ops.gqa_attention_decode(want, kc, vc, ln, out=want), ref)


def test_sequences_that_share_a_cache_they_only_read():
    kc, vc, q = rnd(1, 2000, 2, D, seed=53), rnd(1, 2000, 2, D, seed=54), rnd(3, 4, D, seed=55)
    kc, vc = kc.expand(3, -1, -1, -1), vc.expand(3, -1, -1, -1)
    check(ops.gqa_attention_decode(q, kc, vc, i32([2000, 3, 1500]), rope_theta=0.0), q, kc, vc, [2000, 3, 1500])
    with pytest.raises(ValueError, match="strides of 0"):
        ops.gqa_attention_decode(q, kc, vc, i32([9, 3, 1]), k=rnd(3, 2, D, seed=56), v=rnd(3, 2, D, seed=57))


def test_large_scores_and_far_positions():
    n = 100001
    kc, vc = rnd(1, n, 1, D, seed=12, std=5.0), rnd(1, n, 1, D, seed=13)
    q, k, v = rnd(1, 2, D, seed=14, std=5.0), rnd(1, 1, D, seed=15, std=5.0), rnd(1, 1, D, seed=16)
    o = ops.gqa_attention_decode(q, kc, vc, i32([n]), rope_theta=0.0)
    # fp32 scores of some hundreds (log2 units): off by at most 2^-24 * 128 * sum|q k| ~ 4e-3, and so are the weights
    kk = kc[0].double().expand(n, 2, D)
    ref = torch.einsum("hj,jhd->hd", (torch.einsum("hd,jhd->hj", q[0].double(), kk) / math.sqrt(D)).softmax(-1),
                       vc[0].double().expand(n, 2, D))
    vmax = float(vc.abs().max())
    assert ((o[0].double() - ref).abs() <= 1.01 * 2.0 ** -8 * (ref.abs() + vmax) + 8e-3 * vmax).all()
    ops.gqa_attention_decode(q, kc, vc, i32([n]), k=k, v=v)
    ref = turn(k[0], n - 1, 1e6)
    # an angle reduced in 64 bits is off by 2e-7 radians, times |k| <= 5 * 6
    assert ((kc[0, n - 1].double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 2e-5).all()


def test_offsets_past_32_bits():
    batch, room, hkv = 3, 1 << 20, 8  # 3.2e9 elements of each cache
    kc = torch.empty(batch, room, hkv, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    n = 600
    kc[:, :n], vc[:, :n] = rnd(batch, n, hkv, D, seed=17), rnd(batch, n, hkv, D, seed=18)
    q = rnd(batch, 16, D, seed=19)
    lengths = [n, 0, n - 1]
    check(ops.gqa_attention_decode(q, kc, vc, i32(lengths), rope_theta=0.0), q, kc, vc, lengths)
    k, v = rnd(batch, hkv, D, seed=20), rnd(batch, hkv, D, seed=21)
    kc[2].zero_()
    vc[2].zero_()
    ops.gqa_attention_decode(q, kc, vc, i32([0, 0, room]), k=k, v=v, rope_theta=0.0)
    assert torch.equal(kc[2, -1], k[2]) and torch.equal(vc[2, -1], v[2])


def test_lengths_outside_the_room_are_taken_as_the_nearest():
    kc, vc, q = rnd(3, 40, 1, D, seed=22), rnd(3, 40, 1, D, seed=23), rnd(3, 2, D, seed=24)
    o = ops.gqa_attention_decode(q, kc, vc, i32([41, -1, 1 << 30]), rope_theta=0.0)
    check(o, q, kc, vc, [40, 0, 40])


@pytest.mark.parametrize("room", [256, 512, 4096, 17000])
def test_non_finite_values_that_are_seen(room):
    kc, vc, q = rnd(2, room, 2, D, seed=25), rnd(2, room, 2, D, seed=26), rnd(2, 4, D, seed=27).abs()
    vc[0, 100, 0, 7] = math.inf
    kc[1, 200, 1, 3] = math.nan
    o = ops.gqa_attention_decode(q, kc, vc, i32([room, room]), rope_theta=0.0)
    bad = torch.zeros(2, 4, D, dtype=torch.bool, device="cuda")
    bad[0, :2, 7] = True
    bad[1, 2:] = True
    assert torch.equal(~o.isfinite(), bad)


@pytest.mark.parametrize("room", [256, 3000, 17000])
def test_two_graphs_interleaved_with_growing_lengths(room):
    kc, vc = torch.zeros(2, 2, room, 2, D, dtype=torch.bfloat16, device="cuda").unbind(0)
    q, k, v, ln = rnd(2, 4, D, seed=28), rnd(2, 2, D, seed=29), rnd(2, 2, D, seed=30), i32([100, 200])
    outs = [torch.empty(2, 4, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kc[:, :250], vc[:, :250] = rnd(2, 250, 2, D, seed=31), rnd(2, 250, 2, D, seed=32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        ops.gqa_attention_decode(q, kc, vc, ln, k=k, v=v, out=outs[0])
        for o in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                ops.gqa_attention_decode(q, kc, vc, ln, k=k, v=v, out=o)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(stream)
    for step in range(4):
        q.copy_(rnd(2, 4, D, seed=40 + step))
        ln.copy_(i32([101 + step, 201 + step]))
        graphs[step & 1].replay()
        check(outs[step & 1], q, kc, vc, [101 + step, 201 + step], 1e6)


@pytest.mark.parametrize("room", [700, 17000])
def test_two_streams_at_once(room):
    kc, vc, q = rnd(5, room, 4, D, seed=60), rnd(5, room, 4, D, seed=61), rnd(5, 16, D, seed=62)
    ln, streams = i32([room, 3, 0, 400, 650]), [torch.cuda.Stream() for _ in range(3)]
    want = ops.gqa_attention_decode(q, kc, vc, ln)
    torch.cuda.synchronize()
    outs = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.gqa_attention_decode(q, kc, vc, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("room", [5000, 17000])
def test_same_inputs_same_bits(room):
    kc, vc, q = rnd(3, room, 4, D, seed=33), rnd(3, room, 4, D, seed=34), rnd(3, 16, D, seed=35)
    ln = i32([5000, 1234, 77])
    a = ops.gqa_attention_decode(q, kc, vc, ln, rope_theta=0.0)
    assert torch.equal(a, ops.gqa_attention_decode(q, kc, vc, ln, rope_theta=0.0))


def test_empty_batch():
    e = torch.empty(0, 4, D, dtype=torch.bfloat16, device="cuda")
    c = torch.empty(0, 64, 2, D, dtype=torch.bfloat16, device="cuda")
    assert ops.gqa_attention_decode(e, c, c, i32([])).shape == (0, 4, D)


def test_refusals():
    kc, vc, q, ln = rnd(2, 32, 2, D, seed=36), rnd(2, 32, 2, D, seed=37), rnd(2, 4, D, seed=38), i32([3, 4])
    k = rnd(2, 2, D, seed=39)
    call = ops.gqa_attention_decode
    with pytest.raises(ValueError, match="same batch"):
        call(q[:1], kc, vc, ln)
    with pytest.raises(ValueError, match="int32"):
        call(q, kc, vc, ln.long())
    with pytest.raises(ValueError, match="come together"):
        call(q, kc, vc, ln, k=k)
    with pytest.raises(ValueError, match="contiguous heads"):
        call(q, kc.float(), vc, ln)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        call(rnd(2, 3, D, seed=40), kc, vc, ln)
    with pytest.raises(ValueError, match="multiple of 8"):
        pad = torch.zeros(2, 32, 2 * D + 4, dtype=torch.bfloat16, device="cuda")[..., :2 * D].unflatten(2, (2, D))
        call(q, pad, vc, ln)
    with pytest.raises(ValueError, match="rope_theta"):
        call(q, kc, vc, ln, rope_theta=math.inf)


# a block, a cluster and a split of the device per head; one and several query heads of each kind of tile
@pytest.mark.parametrize("room,lengths", [(200, [1, 0, 200]), (2000, [1, 0, 1999]), (17000, [1, 0, 16999])])
@pytest.mark.parametrize("hq", [4, 24])
@pytest.mark.parametrize("theta", [0.0, 1e6])
def test_scores_that_are_all_minus_infinity(room, lengths, hq, theta):
    """Softmax of nothing but -infinity is NaN; an empty sequence stays 0."""
    kc, vc, q = rnd(3, room, 2, D, seed=70), rnd(3, room, 2, D, seed=71), rnd(3, hq, D, seed=72).abs()
    if theta:  # pair 63 turns by 1e-6 of a position: its first half keeps its sign
        q[..., 127] = 0.0
    kc[:, :, 0, 63] = -math.inf
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), rope_theta=theta)
    for b, n in enumerate(lengths):
        if n == 0:
            assert (o[b] == 0).all()
        else:
            assert o[b, :hq // 2].isnan().all() and o[b, hq // 2:].isfinite().all()


@pytest.mark.parametrize("room,lengths,hq,hkv", [c for c in CASES if sum(c[1])])
@pytest.mark.parametrize("theta", [0.0, 1e6])
def test_precision_of_the_two_part_products(room, lengths, hq, hkv, theta):
    """The bound of queries and weights carried as hi + lo: narrow enough that
    the lo parts, the rotation and the new token have to be there
    (test_attention_bounds_cpu.py plants those mistakes)."""
    batch = len(lengths)
    kc, vc = rnd(batch, room, hkv, D, seed=80), rnd(batch, room, hkv, D, seed=81)
    q, k, v = rnd(batch, hq, D, seed=82), rnd(batch, hkv, D, seed=83), rnd(batch, hkv, D, seed=84)
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), k=k, v=v, rope_theta=theta)
    assert _attention.excess(o, q, kc, vc, lengths, theta) <= 0


@pytest.mark.parametrize("room,lengths,hq,hkv", [c for c in CASES if sum(c[1])])
def test_keys_that_carry_the_weight(room, lengths, hq, hkv):
    """Some thirty keys per sequence, the first, the new one and at least one in
    every part of a split, with nearly all the weight: none may be lost."""
    batch, theta, group = len(lengths), 1e6, hq // hkv
    kc, vc = rnd(batch, room, hkv, D, seed=85), rnd(batch, room, hkv, D, seed=86)
    q, k, v = rnd(batch, hq, D, seed=87), rnd(batch, hkv, D, seed=88), rnd(batch, hkv, D, seed=89)
    for b, n in enumerate(lengths):
        if n:
            _attention.lift(q[b], kc[b, :n], _attention.heavy_keys(n), n - 1, theta)
            for h in range(hkv):  # turned like q, so along it
                x = q[b, h * group].double()
                k[b, h] = (x * ((math.log(n) + 2) * math.sqrt(D) / float(x @ x))).to(k.dtype)
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), k=k, v=v, rope_theta=theta)
    assert _attention.excess(o, q, kc, vc, lengths, theta) <= 0


@pytest.mark.parametrize("room,lengths", [(200, [70, 0, 200]), (2000, [17, 0, 1999]), (17000, [3, 0, 16999])])
@pytest.mark.parametrize("hq", [4, 24])
@pytest.mark.parametrize("theta", [0.0, 1e6])
def test_a_key_of_minus_infinite_score_has_weight_zero(room, lengths, hq, theta):
    kc, vc, q = rnd(3, room, 2, D, seed=73), rnd(3, room, 2, D, seed=74), rnd(3, hq, D, seed=75).abs()
    if theta:  # pair 63 turns by 1e-6 of a position: its first half keeps its sign
        q[..., 127] = 0.0
    keep = torch.ones(room, dtype=torch.bool, device="cuda")
    for j in (0, 16, 150, 1700, 16990):
        if j < room:
            kc[:, j, :, 63], keep[j] = -math.inf, False
    o = ops.gqa_attention_decode(q, kc, vc, i32(lengths), rope_theta=theta)
    for b, n in enumerate(lengths):
        live = keep[:n]
        ref = _attention.definition(q[b], kc[b, :n][live], vc[b, :n][live], n - 1, theta) if n else (0.0, 0.0)
        assert _attention.beyond(o[b], *ref) <= 0


def test_memory_that_is_shared_is_refused_and_views_of_one_buffer_are_not():
    batch, room, hq, hkv = 3, 300, 4, 2
    call, ln = ops.gqa_attention_decode, i32([300, 0, 77])
    buf = rnd(batch, (2 * hq + 2 * hkv) * D, seed=90)
    q, k, v, o = (t.unflatten(1, (-1, D)) for t in buf.split([hq * D, hkv * D, hkv * D, hq * D], 1))
    apart = [rnd(batch, room, hkv, D, seed=91 + i) for i in range(2)]
    want = call(q.clone(), *(c.clone() for c in apart), ln, k=k.clone(), v=v.clone())
    # keys and values side by side in one tensor, by token and by head
    for kv in (torch.stack(apart, 2).unbind(2), torch.stack(apart, 3).unbind(3),
               [c.transpose(1, 2) for c in torch.stack([c.transpose(1, 2) for c in apart], 3).unbind(3)]):
        assert call(q, *kv, ln, k=k, v=v, out=o) is o
        assert torch.equal(o, want)
    kc, vc = apart
    for out in (buf[:, D:(hq + 1) * D].unflatten(1, (-1, D)), q[:, :2]):
        with pytest.raises(ValueError, match="q itself|shape of q"):
            call(q, kc, vc, ln, k=k, v=v, out=out)
    for out in (kc[0, :batch * 2].view(batch, hq, D), buf[:, 2 * hkv * D:4 * hkv * D].unflatten(1, (-1, D))):
        with pytest.raises(ValueError, match="o must not overlap"):
            call(q, kc, vc, ln, k=k, v=v, out=out)
    with pytest.raises(ValueError, match="must be apart"):
        whole = torch.cat([kc, vc], 1)
        call(q, whole[:, :room], whole[:, 1:room + 1], ln, k=k, v=v)
    with pytest.raises(ValueError, match="rows of a cache"):
        call(q, torch.as_strided(kc, (batch, room, hkv, D), (room * D, D, 64, 1)), vc, ln, k=k, v=v)
    with pytest.raises(ValueError, match="caches that take"):
        call(q, kc, vc, ln, k=kc[:, 5], v=v)
    # caches that are only read may be anything
    assert call(q, kc, kc, ln).isfinite().all()
    ops.device_status()
