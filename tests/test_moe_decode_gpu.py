"""The few-token MoE layer on the GPU against its definition in 64 bits.

Tolerance, from the roundings the layer makes: the hidden activations are
rounded to bf16 (2^-8 relative at most), which moves y by at most
2^-8 * sum_r gate_r |W_d| |h|; gate and up sums are fp32, a chain of at most 64
additions per product (each off by 2^-23 of at most sum|w x|, so 2^-17 of it),
which moves h by at most 1.1 |u| dg + |g| du (|silu'| <= 1.1, |silu(g)| <= |g|);
y is rounded to bf16 once (2^-8).  One part in a hundred more is allowed for the
fp32 sums of the second product and the gates."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ennx_b200 import ops  # noqa: E402


def rnd(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def weights(H, E, I, seed):
    return (rnd(E, H, seed=seed, std=1.5 / math.sqrt(H)), rnd(E, 2 * I, H, seed=seed + 1, std=H ** -0.5),
            rnd(E, H, I, seed=seed + 2, std=I ** -0.5))


def routing(x, wr, k):
    logits = x.double() @ wr.double().T
    kept, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    return idx[:, :k], kept[:, :k].softmax(1)


def reference(x, wgu, wd, idx, gate):
    """(y, bound without the output's rounding) of the experts' sum."""
    T, k = idx.shape
    y = torch.zeros(T, wd.shape[1], dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(y)
    for t in range(T):
        for r in range(k):
            e = int(idx[t, r])
            w, xx, d = wgu[e].double(), x[t].double(), wd[e].double()
            both, size = (w @ xx).view(-1, 2, 128), (w.abs() @ xx.abs()).view(-1, 2, 128) * 2.0 ** -17
            g, u = both[:, 0].reshape(-1), both[:, 1].reshape(-1)
            dg, du = size[:, 0].reshape(-1), size[:, 1].reshape(-1)
            h = torch.nn.functional.silu(g) * u
            dh = 2.0 ** -8 * h.abs() + 1.1 * u.abs() * dg + g.abs() * du
            y[t] += gate[t, r] * (d @ h)
            bound[t] += gate[t, r] * (d.abs() @ dh)
    return y, bound


def check(got, x, wgu, wd, idx, gate, residual=None):
    ref, bound = reference(x, wgu, wd, idx, gate)
    if residual is not None:
        ref = ref + residual.double()
    err = (got.double() - ref).abs() - 1.01 * (bound + 2.0 ** -8 * ref.abs()) - 1e-6
    assert err.max() <= 0, float(err.max())


CASES = [
    (1, 256, 8, 2, 128), (1, 2048, 64, 8, 768), (2, 64, 4, 4, 128), (5, 320, 40, 8, 256), (8, 1152, 16, 1, 128),
    (9, 256, 1, 1, 128), (17, 448, 8, 3, 384), (33, 640, 5, 5, 128), (64, 256, 8, 8, 256), (64, 512, 64, 8, 128),
    (40, 2112, 3, 2, 128), (3, 4160, 9, 4, 1152), (64, 128, 256, 8, 128), (7, 2304, 33, 2, 640),
]


@pytest.mark.parametrize("T,H,E,k,I", CASES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_matches_definition(T, H, E, k, I, with_residual):
    x, (wr, wgu, wd) = rnd(T, H, seed=1), weights(H, E, I, 2)
    res = rnd(T, H, seed=5) if with_residual else None
    y, idx, gate = ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res, return_routing=True)
    ridx, rgate = routing(x, wr, k)
    assert torch.equal(idx.long(), ridx)
    torch.testing.assert_close(gate.double(), rgate, rtol=2e-5, atol=0)
    check(y, x, wgu, wd, ridx, rgate, res)
    assert torch.equal(ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res), y)


def test_agrees_with_the_full_layer():
    T, H, E, k, I = 48, 1024, 16, 8, 256
    x, (wr, wgu, wd), res = rnd(T, H, seed=6), weights(H, E, I, 7), rnd(T, H, seed=10)
    y, idx, gate = ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res, return_routing=True)
    full, fidx, fgate = ops.moe_layer(x, wr, wgu, wd, k, residual=res, return_routing=True)
    assert torch.equal(idx, fidx)
    torch.testing.assert_close(gate, fgate, rtol=1e-5, atol=1e-6)
    # the full layer also rounds every expert's output to bf16
    ref, bound = reference(x, wgu, wd, idx, gate.double())
    spread = sum((gate[:, r, None].double() * wd[idx[:, r].long()].double().abs().sum(2)) for r in range(k))
    assert ((y.double() - full.double()).abs() <= 2.02 * (bound + 2.0 ** -8 * (ref + res.double()).abs()) +
            2.0 ** -8 * spread * float(x.float().abs().max()) + 1e-6).all()


def test_all_tokens_pick_the_same_experts():
    T, H, E, k, I = 64, 256, 16, 2, 128
    x, (wr, wgu, wd) = rnd(1, H, seed=11).expand(T, H).contiguous(), weights(H, E, I, 12)
    y, idx, _ = ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True)
    assert (idx == idx[0]).all() and (y == y[0]).all()
    ridx, rgate = routing(x, wr, k)
    check(y, x, wgu, wd, ridx, rgate)


@pytest.mark.parametrize("T,E,k,I", [(64, 16, 2, 640), (64, 40, 4, 128), (17, 12, 1, 256), (49, 9, 3, 384)])
def test_uneven_routing(T, E, k, I):
    """Experts from one token to nearly all, so groups of tokens from one to four side by side."""
    H = 256
    x, (wr, wgu, wd) = rnd(T, H, seed=27), weights(H, E, I, 28)
    pull = rnd(1, H, seed=31)
    x = (x.float() + pull.float() * torch.linspace(0, 2, T, device="cuda")[:, None]).to(torch.bfloat16)
    wr[E // 2] += pull[0] / 8
    wr[E - 1] += pull[0] / 16
    y, idx, gate = ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True)
    ridx, rgate = routing(x, wr, k)
    assert torch.equal(idx.long(), ridx)
    check(y, x, wgu, wd, ridx, rgate)


@pytest.mark.parametrize("E,k", [(16, 8), (200, 8), (8, 8), (33, 1)])
def test_ties_keep_the_lower_index(E, k):
    H, I = 256, 128
    _, wgu, wd = weights(H, E, I, 15)
    wr = rnd(1, H, seed=18).repeat(E, 1)
    _, idx, gate = ops.moe_layer_decode(rnd(9, H, seed=19), wr, wgu, wd, k, return_routing=True)
    assert idx.tolist() == [list(range(k))] * 9
    torch.testing.assert_close(gate, torch.full_like(gate, 1.0 / k), rtol=1e-6, atol=0)


def test_a_bad_token_or_expert_stays_with_its_own():
    T, H, E, k, I = 12, 256, 8, 2, 128
    x, (wr, wgu, wd) = rnd(T, H, seed=20), weights(H, E, I, 21)
    clean = ops.moe_layer_decode(x, wr, wgu, wd, k)
    ridx, _ = routing(x, wr, k)
    bad = x.clone()
    bad[5, 7] = math.nan
    y, idx, _ = ops.moe_layer_decode(bad, wr, wgu, wd, k, return_routing=True)
    others = [t for t in range(T) if t != 5]
    assert torch.equal(y[others], clean[others]) and y[5].isnan().all()
    assert torch.equal(idx[others].long(), ridx[others]) and idx[5].min() >= 0 and idx[5].max() < E
    assert len(set(idx[5].tolist())) == k
    e = int(ridx[0, 0])
    wgu[e, 3] = math.inf
    y = ops.moe_layer_decode(x, wr, wgu, wd, k)
    uses = (ridx == e).any(1)
    assert torch.equal(y[~uses], clean[~uses]) and not y[uses].isfinite().any()


@pytest.mark.parametrize("T", [3, 12, 40])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_bad_down_weights_reach_only_the_tokens_of_their_expert(T, bad):
    H, E, k, I = 256, 8, 2, 128
    x, (wr, wgu, wd) = rnd(T, H, seed=24), weights(H, E, I, 25)
    clean, idx, _ = ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True)
    e = int(idx[0, 0])
    wd[e, 3:, ::5] = bad
    y = ops.moe_layer_decode(x, wr, wgu, wd, k)
    touched = (idx == e).any(1)
    assert torch.equal(y[~touched], clean[~touched]) and torch.equal(y[:, :3], clean[:, :3])
    assert not y[touched][:, 3:].isfinite().any()


def test_residual_in_place_and_other_stream_and_graph():
    T, H, E, k, I = 4, 512, 16, 4, 128
    x, (wr, wgu, wd) = rnd(T, H, seed=24), weights(H, E, I, 25)
    res = rnd(T, H, seed=28)
    want = ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res)
    inplace = res.clone()
    assert ops.moe_layer_decode(x, wr, wgu, wd, k, residual=inplace, out=inplace) is inplace
    assert torch.equal(inplace, want)
    out, out2 = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res, out=out)
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        for g, o in zip(graphs, (out, out2)):
            with torch.cuda.graph(g, stream=stream):
                ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res, out=o)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(3):
        x.copy_(rnd(T, H, seed=30 + seed))
        for g in graphs:
            g.replay()
        want = ops.moe_layer_decode(x, wr, wgu, wd, k, residual=res)
        assert torch.equal(out, want) and torch.equal(out2, want)


def test_two_streams_at_once():
    T, H, E, k, I = 8, 1024, 32, 8, 256
    xs = [rnd(T, H, seed=40), rnd(T, H, seed=41)]
    wr, wgu, wd = weights(H, E, I, 42)
    want = [ops.moe_layer_decode(x, wr, wgu, wd, k) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.moe_layer_decode(xs[i], wr, wgu, wd, k))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_no_tokens():
    wr, wgu, wd = weights(256, 8, 128, 50)
    y = ops.moe_layer_decode(torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), wr, wgu, wd, 2)
    assert y.shape == (0, 256)


def test_refusals():
    x, (wr, wgu, wd) = rnd(4, 256, seed=60), weights(256, 8, 128, 61)
    call = ops.moe_layer_decode
    with pytest.raises(Exception, match="at most 64 tokens"):
        call(rnd(65, 256, seed=64), wr, wgu, wd, 2)
    with pytest.raises(ValueError, match="top_k"):
        call(x, wr, wgu, wd, 9)
    with pytest.raises(ValueError, match="top_k"):
        call(x, wr, wgu, wd, 0)
    with pytest.raises(ValueError, match="weights must be"):
        call(x, wr, wgu, wd.transpose(1, 2), 2)
    with pytest.raises(ValueError, match="contiguous bfloat16"):
        call(x.float(), wr, wgu, wd, 2)
    with pytest.raises(ValueError, match="contiguous bfloat16"):
        call(x, wr, wgu, wd, 2, residual=rnd(4, 512, seed=65)[:, ::2])
    with pytest.raises(ValueError, match="shape of x"):
        call(x, wr, wgu, wd, 2, residual=x[:2])
    with pytest.raises(ValueError, match="CUDA"):
        call(x.cpu(), wr, wgu, wd, 2)


@pytest.mark.parametrize("T,H,E,k", [(1, 64, 1, 1), (8, 64, 1, 1), (64, 64, 3, 2), (9, 64, 9, 8)])
def test_router_whose_blocks_have_next_to_nothing_to_do(T, H, E, k):
    """A block of the router stores logits into other blocks' shared memory soon
    after its start here, or has no expert at all and only receives them."""
    x, (wr, wgu, wd) = rnd(T, H, seed=70), weights(H, E, 128, 71)
    y, idx, gate = ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True)
    ridx, rgate = routing(x, wr, k)
    assert torch.equal(idx.long(), ridx)
    check(y, x, wgu, wd, ridx, rgate)
    runs = [ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True) for _ in range(200)]
    assert all(torch.equal(a, y) and torch.equal(b, idx) and torch.equal(c, gate) for a, b, c in runs)
    ops.device_status()


def test_out_that_shares_memory_is_refused():
    T, H, E, k, I = 4, 256, 8, 2, 128
    buf, (wr, wgu, wd) = rnd(5 * T, H, seed=80), weights(H, E, I, 81)
    x, res, call = buf[:T], buf[T:2 * T], ops.moe_layer_decode
    for out in (x, buf[1:T + 1], wr[:T], wgu[0, :T]):
        with pytest.raises(ValueError, match="must not overlap"):
            call(x, wr, wgu, wd, k, residual=res, out=out)
    with pytest.raises(ValueError, match="must not overlap"):
        call(x, wr, wgu, wd, k, residual=res, out=buf[T + 1:2 * T + 1])
    want = call(x, wr, wgu, wd, k, residual=res)
    assert torch.equal(call(x, wr, wgu, wd, k, residual=res, out=buf[2 * T:3 * T]), want)
    assert torch.equal(call(x, wr, wgu, wd, k, residual=x), call(x, wr, wgu, wd, k, residual=x.clone()))
    assert torch.equal(call(x, wr, wgu, wd, k, residual=res, out=res), want)


@pytest.mark.parametrize("T", [2, 20])
def test_weight_offsets_past_32_bits(T):
    H, E, k, I = 8192, 160, 2, 1024  # 2.7e9 elements of gate and up, 1.3e9 of down
    g = torch.Generator(device="cuda").manual_seed(90)
    wgu = torch.randn(E, 2 * I, H, generator=g, device="cuda", dtype=torch.bfloat16).mul_(H ** -0.5)
    wd = torch.randn(E, H, I, generator=g, device="cuda", dtype=torch.bfloat16).mul_(I ** -0.5)
    x, wr = rnd(T, H, seed=91), rnd(E, H, seed=92, std=1.5 / H ** 0.5)
    wr[E - 1] = wr[E - 1] + x[0] / 32  # the last expert is picked
    y, idx, _ = ops.moe_layer_decode(x, wr, wgu, wd, k, return_routing=True)
    ridx, rgate = routing(x, wr, k)
    assert torch.equal(idx.long(), ridx) and int(ridx.max()) == E - 1
    check(y, x, wgu, wd, ridx, rgate)
