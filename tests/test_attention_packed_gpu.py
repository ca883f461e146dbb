"""Attention over packed prompts on the GPU against its definition in 64 bits.

Tolerance: the output is rounded to bf16 once (2^-8 of a value at most), and
P is rounded to bf16 before P V (each weight off by at most 2^-8 relative, so
the sum by at most 2^-8 * sum |p v| <= 2^-8 * max |v|).  Together
|got - ref| <= 2^-8 |ref| + 2^-8 max|v|, and fp32 sums add far less; the test
allows one part in a thousand more."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ennx_b200 import ops  # noqa: E402

D = 128


def rnd(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def starts(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def turned(x, lengths, theta):
    """RoPE of packed x [rows, heads, 128] in 64 bits."""
    pos = torch.cat([torch.arange(n) for n in lengths]).double().cuda()
    inv = theta ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    a = pos[:, None] * inv
    c, s = a.cos()[:, None], a.sin()[:, None]
    x1, x2 = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def reference(q, k, v, lengths):
    out, at = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0
    group = q.shape[1] // k.shape[1]
    for n in lengths:
        r = slice(at, at + n)
        at += n
        kk, vv = k[r].double().repeat_interleave(group, 1), v[r].double().repeat_interleave(group, 1)
        a = torch.einsum("ihd,jhd->hij", q[r].double(), kk) / math.sqrt(D)
        a.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        out[r] = torch.einsum("hij,jhd->ihd", a.softmax(-1), vv)
    return out


def close(got, ref, vmax, extra=0.0):
    err = (got.double() - ref).abs() - (1.001 * 2.0 ** -8 * (ref.abs() + vmax) + extra)
    assert err.max() <= 0, float(err.max())


CASES = [
    ([1], 1, 1), ([2, 1, 1], 2, 1), ([128], 4, 4), ([127, 129], 4, 2), ([256, 1, 255], 4, 1), ([5] * 60, 8, 2),
    ([1] * 300, 2, 1), ([0, 7, 0, 0, 300, 0], 4, 1), ([700, 3, 40, 513], 16, 4), ([1, 1300], 3, 1),
    ([31, 97, 1, 129, 64, 512, 2], 6, 2),
]


@pytest.mark.parametrize("lengths,hq,hkv", CASES)
def test_matches_definition(lengths, hq, hkv):
    rows = sum(lengths)
    q, k, v = rnd(rows, hq, D, seed=1), rnd(rows, hkv, D, seed=2), rnd(rows, hkv, D, seed=3)
    q0, k0 = q.clone(), k.clone()
    o = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    ops.device_status()
    assert torch.equal(q, q0) and torch.equal(k, k0)
    close(o, reference(q, k, v, lengths), float(v.float().abs().max()))


def test_large_scores():
    # scores of some hundreds: the running maximum moves by more than the lazy rescale's 2^8 many times
    lengths = [300, 900]
    q, k, v = rnd(1200, 4, D, seed=4, std=6.0), rnd(1200, 2, D, seed=5, std=6.0), rnd(1200, 2, D, seed=6)
    o = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    # an fp32 score of a few hundred (in units of log2) is off by up to 2^-24 * 128 * sum|q k| ~ 2e-3 at most,
    # which moves a weight by that much relative to itself
    close(o, reference(q, k, v, lengths), float(v.float().abs().max()), extra=4e-3 * float(v.float().abs().max()))


def test_rope_positions_restart_with_each_sequence():
    lengths = [200, 0, 1, 333]
    rows = sum(lengths)
    q, k, v = rnd(rows, 4, D, seed=7), rnd(rows, 2, D, seed=8), rnd(rows, 2, D, seed=9)
    rq, rk = turned(q, lengths, 1e6), turned(k, lengths, 1e6)
    o = ops.gqa_attention_packed(q, k, v, starts(lengths))
    for got, ref in ((q, rq), (k, rk)):  # one rounding to bf16 of an fp32 rotation
        assert ((got.double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 1e-5).all()
    close(o, reference(q, k, v, lengths), float(v.float().abs().max()))


def test_columns_of_a_fused_projection_and_rows_behind_the_last_sequence():
    lengths, spare, hq, hkv = [190, 77], 200, 4, 2
    rows = sum(lengths) + spare
    ld = (hq + 2 * hkv) * D + 16
    buf = rnd(rows, ld, seed=10)
    live = sum(lengths)
    buf[live:] = math.nan
    buf[live + 1:, ::3] = math.inf
    before = buf.clone()
    q = buf[:, :hq * D].unflatten(1, (hq, D))
    k = buf[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D))
    v = buf[:, (hq + hkv) * D:(hq + 2 * hkv) * D].unflatten(1, (hkv, D))
    out = torch.full((rows, hq * D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    o = out[:, :hq * D].unflatten(1, (hq, D))
    ref = reference(q[:live], k[:live], v[:live], lengths)
    ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0, out=o)
    close(o[:live], ref, float(v[:live].float().abs().max()))
    assert (out[live:] == 7.0).all() and (out[:, hq * D:] == 7.0).all()
    assert torch.equal(buf.view(torch.int16), before.view(torch.int16))
    ops.gqa_attention_packed(q, k, v, starts(lengths), out=o)  # rotates the live rows only
    assert torch.equal(buf[live:].view(torch.int16), before[live:].view(torch.int16))
    assert torch.equal(buf[:, (hq + hkv) * D:].view(torch.int16), before[:, (hq + hkv) * D:].view(torch.int16))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_values_reach_only_the_rows_that_see_them(bad):
    lengths = [100, 200, 60]
    q, k, v = rnd(360, 4, D, seed=11), rnd(360, 2, D, seed=12), rnd(360, 2, D, seed=13)
    clean = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    v[150, 1, 5] = bad      # sequence 1, its row 50
    k[330, 0, 9] = math.nan  # sequence 2, its row 30
    o = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    touched = torch.zeros(360, 4, D, dtype=torch.bool, device="cuda")
    touched[150:300, 2:, 5] = True
    touched[330:360, :2, :] = True
    assert torch.equal(o.isfinite(), ~touched)
    # rows that the check recomputed carry fp32 weights, the others bf16 ones: both within the bound of the definition
    vv = v.clone()
    vv[150, 1, 5] = 0
    ref = reference(q[:330], k[:330], vv[:330], [100, 200, 30])
    assert float((o[:330].double() - ref)[~touched[:330]].abs().max()) <= 2 * 2.0 ** -8 * float(vv.float().abs().max())
    assert torch.equal(o[:100], clean[:100])


def test_infinite_key_scores():
    # a visible score of +inf makes its rows NaN, as softmax does; other sequences stay whole
    q, k, v = rnd(80, 1, D, seed=14).abs(), rnd(80, 1, D, seed=15), rnd(80, 1, D, seed=16)
    k[50, 0, 3] = math.inf
    o = ops.gqa_attention_packed(q, k, v, starts([40, 40]), rope_theta=0.0)
    assert o[:50].isfinite().all() and o[50:].isnan().all()


def test_replayed_graph_with_other_lengths_and_a_side_stream():
    rows, hq, hkv = 512, 4, 2
    q, k, v = rnd(rows, hq, D, seed=17), rnd(rows, hkv, D, seed=18), rnd(rows, hkv, D, seed=19)
    cu = starts([300, 212])
    out = torch.empty(rows, hq, D, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    vmax = float(v.float().abs().max())
    for lengths in ([300, 212], [1, 511], [17, 200]):
        cu.copy_(starts(lengths))
        graph.replay()
        n = sum(lengths)
        close(out[:n], reference(q[:n], k[:n], v[:n], lengths), vmax)


def test_captured_with_the_rotation_and_many_items():
    # more blocks than the device holds at once, q and k rotated in front, fresh operands at every replay
    lengths, hq, hkv = [1500, 1, 700, 0, 1647, 252], 16, 4
    rows = sum(lengths)
    q, k, v = rnd(rows, hq, D, seed=30), rnd(rows, hkv, D, seed=31), rnd(rows, hkv, D, seed=32)
    qs, ks, cu = q.clone(), k.clone(), starts(lengths)
    want = ops.gqa_attention_packed(qs, ks, v, cu)
    assert ((want.double() - reference(qs, ks, v, lengths)).abs() <= 1.001 * 2.0 ** -8 * 2 * float(v.float().abs().max())).all()
    graph, q1, k1 = torch.cuda.CUDAGraph(), torch.empty_like(q), torch.empty_like(k)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        q1.copy_(q)
        k1.copy_(k)
        got = ops.gqa_attention_packed(q1, k1, v, cu)
    for _ in range(3):
        graph.replay()
        assert torch.equal(got, want) and torch.equal(q1, qs) and torch.equal(k1, ks)


def test_two_streams_at_once():
    lengths = [900, 37, 2200]
    rows, one, two = sum(lengths), torch.cuda.Stream(), torch.cuda.Stream()
    q, k, v = rnd(rows, 16, D, seed=33), rnd(rows, 4, D, seed=34), rnd(rows, 4, D, seed=35)
    cu = starts(lengths)
    want = ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0)
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in (one, two):
            with torch.cuda.stream(s):
                outs.append(ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_same_inputs_same_bits():
    lengths = [900, 124]
    q, k, v = rnd(1024, 8, D, seed=20), rnd(1024, 2, D, seed=21), rnd(1024, 2, D, seed=22)
    a = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    b = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    assert torch.equal(a, b)


def test_no_rows():
    e = torch.empty(0, 4, D, dtype=torch.bfloat16, device="cuda")
    o = ops.gqa_attention_packed(e, e[:, :2], e[:, :2], starts([0, 0]))
    assert o.shape == (0, 4, D)


def test_refusals():
    q, k, v, cu = rnd(8, 4, D, seed=23), rnd(8, 2, D, seed=24), rnd(8, 2, D, seed=25), starts([8])
    call = ops.gqa_attention_packed
    with pytest.raises(ValueError, match="bfloat16"):
        call(q.half(), k, v, cu)
    with pytest.raises(ValueError, match="same rows"):
        call(q, k[:7], v[:7], cu)
    with pytest.raises(ValueError, match="int32"):
        call(q, k, v, cu.long())
    with pytest.raises(ValueError, match="multiple of Hkv"):
        call(q[:, :3], k, v, cu)
    with pytest.raises(ValueError, match="contiguous within a row"):
        call(q[:, ::2], k, v, cu)
    with pytest.raises(ValueError, match="rope_theta"):
        call(q, k, v, cu, rope_theta=-1.0)
    odd = torch.zeros(8 * 4 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 4, D)
    with pytest.raises(ValueError, match="16-byte aligned"):
        call(odd, k, v, cu)
    with pytest.raises(ValueError, match="CUDA"):
        call(q.cpu(), k, v, cu)


def test_rows_whose_visible_scores_are_all_minus_infinity():
    """Softmax of nothing but -infinity is NaN; a row that sees one other score is what that score says."""
    lengths = [40, 300, 7, 129]
    q, k, v = rnd(476, 4, D, seed=40).abs(), rnd(476, 2, D, seed=41), rnd(476, 2, D, seed=42)
    k[0, 0, 3] = -math.inf        # the first row of sequence 0 sees nothing else
    k[40:240, 1, 9] = -math.inf   # rows 0 .. 199 of sequence 1, over a tile's end
    k[347:, :, 127] = -math.inf   # all of sequence 3
    o = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    lost = torch.zeros(476, 4, dtype=torch.bool, device="cuda")
    lost[0, :2] = True
    lost[40:240, 2:] = True
    lost[347:] = True
    ref = reference(q, k, v, lengths)
    assert torch.equal(ref.isnan(), lost[:, :, None].expand_as(ref))
    assert torch.equal(o.isnan(), ref.isnan())
    close(o[~lost], ref[~lost], float(v.float().abs().max()))
    ops.device_status()


def test_out_that_shares_memory_is_refused_and_columns_beside_are_not():
    hq, hkv, rows = 4, 2, 300
    buf = rnd(rows, (2 * hq + 2 * hkv) * D, seed=50)
    q, k, v, o = (t.unflatten(1, (-1, D)) for t in buf.split([hq * D, hkv * D, hkv * D, hq * D], 1))
    cu, call = starts([100, 200]), ops.gqa_attention_packed
    want = call(q.clone(), k.clone(), v.clone(), cu)
    for out in (q, buf[:, D:(hq + 1) * D].unflatten(1, (-1, D)), buf[:, 2 * hkv * D:(2 * hkv + hq) * D].unflatten(1, (-1, D))):
        with pytest.raises(ValueError, match="must not overlap"):
            call(q, k, v, cu, out=out)
    with pytest.raises(ValueError, match="in place"):
        call(q, k, buf[:, (hq + 1) * D:(hq + 1 + hkv) * D].unflatten(1, (-1, D)), cu)
    # the same memory twice is fine where nothing is written to it
    call(q, k, k, cu, rope_theta=0.0)
    call(q, q[:, :hkv], k, cu, rope_theta=0.0)
    assert call(q, k, v, cu, out=o) is o
    assert torch.equal(o, want)


def lasts(call, runs=3):
    """Milliseconds of a call, the best of some runs."""
    best = math.inf
    for _ in range(runs):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def test_bad_keys_at_the_start_of_a_long_prompt_cost_no_recomputation():
    rows, hq, hkv = 16384, 16, 4
    q, k, v, cu = rnd(rows, hq, D, seed=60), rnd(rows, hkv, D, seed=61), rnd(rows, hkv, D, seed=62), starts([rows])

    def call():
        return ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0)

    want = call()
    clean = lasts(call)
    for bad in (math.nan, math.inf):
        k[0, :2, 3] = bad
        o = call()
        if bad != bad:
            assert o[:, :8].isnan().all()
        else:  # a score of -infinity leaves its row as the others have it, one of +infinity makes it NaN
            assert torch.equal(o[:, :8].isnan(), (q[:, :8, 3] > 0)[..., None].expand(-1, -1, D) | (torch.arange(rows, device="cuda") == 0)[:, None, None])
        assert torch.equal(o[:, 8:], want[:, 8:])
        assert lasts(call) < 4 * clean
    ops.device_status()


def test_bad_values_at_the_start_of_a_long_prompt_cost_no_recomputation():
    rows, hq, hkv = 16384, 16, 4
    q, k, v, cu = rnd(rows, hq, D, seed=63), rnd(rows, hkv, D, seed=64), rnd(rows, hkv, D, seed=65), starts([rows])

    def call():
        return ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0)

    want = call()
    clean = lasts(call)
    v[0, 0, 5], v[0, 1, 6], v[1000, 3] = math.nan, math.inf, math.nan
    o = call()
    assert o[:, :4, 5].isnan().all() and (o[:, 4:8, 6] == math.inf).all() and o[1000:, 12:].isnan().all()
    same = torch.ones_like(o, dtype=torch.bool)
    same[:, :4, 5] = same[:, 4:8, 6] = same[896:, 12:] = False
    assert torch.equal(o[same], want[same])
    # the rows of its tile before the bad one are recomputed, with weights of fp32
    assert ((o[896:1000, 12:].double() - want[896:1000, 12:].double()).abs() <= 4 * 2.0 ** -8 * 5).all()
    assert lasts(call) < 20 * clean
    ops.device_status()


@pytest.mark.parametrize("many", [3, 60])
def test_bad_values_anywhere(many):
    """Infinities and NaN at random places: each reaches its column of the rows that see it, and nothing else."""
    lengths, hq, hkv = [5, 130, 0, 1, 300, 77, 513], 4, 2
    rows = sum(lengths)
    q, k, v = rnd(rows, hq, D, seed=66), rnd(rows, hkv, D, seed=67), rnd(rows, hkv, D, seed=68)
    g = torch.Generator().manual_seed(69)
    sign = torch.zeros(3, rows, hkv, D, dtype=torch.bool, device="cuda")  # +inf, -inf, NaN
    for _ in range(many):
        at = [int(torch.randint(n, (1,), generator=g)) for n in (3, rows, hkv, D)]
        sign[tuple(at)] = True
    finite = v.masked_fill(sign.any(0), 0.0)
    for s, value in zip(sign, (math.inf, -math.inf, math.nan)):
        v[s] = value
    seq = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()
    visible = ((seq[:, None] == seq) & (torch.arange(rows).cuda()[:, None] >= torch.arange(rows).cuda())).float()
    kinds = torch.stack([v == math.inf, v == -math.inf, v.isnan()])
    sees = (torch.einsum("ij,cjhd->cihd", visible, kinds.float()) > 0).repeat_interleave(hq // hkv, 2)
    nan = sees[2] | (sees[0] & sees[1])
    o = ops.gqa_attention_packed(q, k, v, starts(lengths), rope_theta=0.0)
    assert torch.equal(o.isnan(), nan)
    assert torch.equal(o == math.inf, sees[0] & ~nan) and torch.equal(o == -math.inf, sees[1] & ~nan)
    clean = ~sees.any(0)
    err = (o.double() - reference(q, k, finite, lengths)).abs()[clean]
    # a weight of a value that counts as 0 here is part of the sum in both
    assert float(err.max()) <= 1.001 * 2.0 ** -8 * 2 * float(finite.float().abs().max())
    ops.device_status()


def test_values_near_the_end_of_the_range():
    # the second score is 7 doublings above the first, within the lazy rescale's 8: the product with a weight of 2^7 is no number
    q, k, v = (torch.zeros(2, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    q[:, 0, 0], k[1, 0, 0] = 7.0, 7.0 * math.log(2) * math.sqrt(D) / 7.0
    v[:, 0, 3], v[:, 0, 4] = 1e37, -1e37
    v[:, 0, 5] = 1.0
    o = ops.gqa_attention_packed(q, k, v, starts([2]), rope_theta=0.0)
    ref = reference(q, k, v, [2])
    assert ((o.double() - ref).abs() <= 2.01 * 2.0 ** -8 * ref.abs()).all()


def test_a_long_recomputation_ends_before_the_waits_for_it():
    """A bad last value: the rows of its tile walk the whole prompt one after
    another while every other role waits (3 s at 50000 rows; the walk takes 0.3)."""
    rows = 50000
    q, k, v, cu = rnd(rows, 2, D, seed=70), rnd(rows, 1, D, seed=71), rnd(rows, 1, D, seed=72), starts([rows])
    want = ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0)
    v[-1, 0, 9] = math.nan
    o = ops.gqa_attention_packed(q, k, v, cu, rope_theta=0.0)
    ops.device_status()
    assert o[-1, :, 9].isnan().all() and o[:-1].isfinite().all()
    first = (rows - 1) // 128 * 128
    assert torch.equal(o[:first], want[:first])
    assert ((o[first:-1].double() - want[first:-1].double()).abs() <= 4 * 2.0 ** -8 * 5).all()


@pytest.mark.parametrize("lengths", [[0] * 300 + [70, 0, 129] + [0] * 300, [0] * 40 + [1] + [0] * 40, [0] * 500])
def test_many_empty_sequences_at_both_ends_with_the_rotation(lengths):
    rows = sum(lengths) + 9
    q, k, v = rnd(rows, 4, D, seed=73), rnd(rows, 2, D, seed=74), rnd(rows, 2, D, seed=75)
    q0, k0, out = q.clone(), k.clone(), torch.full((rows, 4, D), 3.0, dtype=torch.bfloat16, device="cuda")
    live = sum(lengths)
    ops.gqa_attention_packed(q, k, v, starts(lengths), out=out)
    assert (out[live:] == 3.0).all() and torch.equal(q[live:], q0[live:]) and torch.equal(k[live:], k0[live:])
    if live:
        for got, before in ((q, q0), (k, k0)):
            ref = turned(before[:live], lengths, 1e6)
            assert ((got[:live].double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 1e-5).all()
        close(out[:live], reference(q[:live], k[:live], v[:live], lengths), float(v.float().abs().max()))
    ops.device_status()


def test_offsets_past_32_bits():
    hq, hkv, n = 16, 4, 997
    count = (1 << 31) // (n * hq * D) + 20  # 2.2e9 elements of q and of the output
    rows = n * count
    g = torch.Generator(device="cuda").manual_seed(80)
    q, k, v = (torch.randn(rows, h, D, generator=g, device="cuda", dtype=torch.bfloat16) for h in (hq, hkv, hkv))
    last = slice(rows - 3 * n, rows)
    rq, rk = (turned(x[last], [n] * 3, 1e6) for x in (q, k))
    o = ops.gqa_attention_packed(q, k, v, starts([n] * count))
    for got, ref in ((q[last], rq), (k[last], rk)):
        assert ((got.double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 1e-5).all()
    close(o[last], reference(q[last], k[last], v[last], [n] * 3), float(v[last].float().abs().max()))
    v[-40, 1, 7] = math.nan  # and where rows are computed again
    o = ops.gqa_attention_packed(q, k, v, starts([n] * count), rope_theta=0.0)
    assert o[-40:, 4:8, 7].isnan().all() and int((~o[last].isfinite()).sum()) == 40 * 4
    ops.device_status()
