"""The serving operators as a GQA-MoE layer uses them: packed prompts fill a
cache, then tokens follow one at a time (fused packed projection, cache
attention, packed output projection, few-token MoE), eagerly and as a replayed
graph.

Each operator is held against its 64-bit definition on the inputs that its
predecessors left, with the tolerance its own tests derive."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import _attention  # noqa: E402
import test_attention_decode_gpu as cached  # noqa: E402
import test_attention_packed_gpu as prompts  # noqa: E402
import test_moe_decode_gpu as moe  # noqa: E402
import test_packed_decode_gpu as packed  # noqa: E402

from ennx_b200 import ops  # noqa: E402

D, THETA = 128, 1e6
rnd = prompts.rnd


class Layer:
    def __init__(self, hidden, hq, hkv, experts, top_k, width, lengths, room):
        self.hq, self.hkv, self.top_k, self.room = hq, hkv, top_k, room
        self.qkv = packed.make(hidden, (hq + 2 * hkv) * D, 4, 64, seed=1)
        self.proj = packed.make(hq * D, hidden, 8, 32, seed=2)
        self.norms = rnd(2, hidden, seed=3)
        self.wr, self.wgu, self.wd = moe.weights(hidden, experts, width, seed=4)
        self.kc = torch.full((len(lengths), room, hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.vc = self.kc.clone()
        self.lengths = cached.i32(lengths)

    def split(self, fused):
        a, b = self.hq * D, (self.hq + self.hkv) * D
        return [t.unflatten(1, (-1, D)) for t in (fused[:, :a], fused[:, a:b], fused[:, b:])]

    def prompt(self, x, lengths):
        q, k, v = self.split(ops.packed_linear(ops.rmsnorm(x, self.norms[0]), *self.qkv))
        q0, k0 = q.clone(), k.clone()
        o = ops.gqa_attention_packed(q, k, v, prompts.starts(lengths), THETA)
        at = 0
        for b, n in enumerate(lengths):
            self.kc[b, :n], self.vc[b, :n] = k[at:at + n], v[at:at + n]
            at += n
        return q0, k0, q, k, v, o

    def token(self, x):
        """One more token of each sequence; every intermediate, the layer's output last."""
        self.lengths.add_(1)
        h = ops.rmsnorm(x, self.norms[0])
        fused = ops.packed_linear_decode(h, *self.qkv)
        q, k, v = self.split(fused)
        o = ops.gqa_attention_decode(q, self.kc, self.vc, self.lengths, k=k, v=v, rope_theta=THETA)
        a = ops.packed_linear_decode(o.flatten(1), *self.proj)
        mid = x + a
        m = ops.rmsnorm(mid, self.norms[1])
        y, idx, gate = ops.moe_layer_decode(m, self.wr, self.wgu, self.wd, self.top_k, residual=mid, return_routing=True)
        return h, fused, o, a, mid, m, idx, gate, y


@pytest.mark.parametrize("room", [400, 1500, 17000])  # clusters of blocks per head; split over the device
def test_prompt_then_tokens(room):
    hidden, lengths = 512, [130, 0, 33, 300, 1]
    layer = Layer(hidden, 4, 2, 8, 3, 128, lengths, room)
    q0, k0, q, k, v, o = layer.prompt(rnd(sum(lengths), hidden, seed=7), lengths)
    for got, before in ((q, q0), (k, k0)):  # one rounding to bf16 of an fp32 rotation
        ref = prompts.turned(before, lengths, THETA)
        assert ((got.double() - ref).abs() <= 1.01 * 2.0 ** -8 * ref.abs() + 1e-5).all()
    prompts.close(o, prompts.reference(q, k, v, lengths), float(v.abs().max()))
    x = rnd(len(lengths), hidden, seed=8)
    for step in range(3):
        now = [n + step + 1 for n in lengths]
        h, fused, o, a, mid, m, idx, gate, y = layer.token(x)
        packed.check(fused, h, *layer.qkv)
        q, _, v = layer.split(fused)
        cached.check(o, q, layer.kc, layer.vc, now, THETA)
        for b, n in enumerate(now):
            assert torch.equal(layer.vc[b, n - 1], v[b]) and layer.kc[b, n:].isnan().all()
        packed.check(a, o.flatten(1), *layer.proj)
        moe.check(y, m, layer.wgu, layer.wd, idx.long(), gate.double(), mid)
        x = y
    ops.device_status()


def test_the_last_token_of_a_prompt_is_what_a_token_step_gives():
    """The same keys and values either way, so the outputs differ by the two
    tolerances against the definition: the prompt's pass turns q to bf16."""
    lengths, hq, hkv = [200, 2, 1, 77], 4, 2
    q, k, v = rnd(sum(lengths), hq, D, seed=9), rnd(sum(lengths), hkv, D, seed=10), rnd(sum(lengths), hkv, D, seed=11)
    last = (prompts.starts(lengths)[1:] - 1).long()
    qt, kt, vt = q[last].clone(), k[last].clone(), v[last].clone()
    o = ops.gqa_attention_packed(q, k, v, prompts.starts(lengths), THETA)
    kc = torch.zeros(len(lengths), 256, hkv, D, dtype=torch.bfloat16, device="cuda")
    vc, at = torch.zeros_like(kc), 0
    for b, n in enumerate(lengths):
        kc[b, :n - 1], vc[b, :n - 1] = k[at:at + n - 1], v[at:at + n - 1]
        at += n
    got = ops.gqa_attention_decode(qt, kc, vc, cached.i32(lengths), k=kt, v=vt, rope_theta=THETA)
    for b, n in enumerate(lengths):
        assert torch.equal(kc[b, n - 1], k[last[b]]) and torch.equal(vc[b, n - 1], v[last[b]])
    cached.check(o[last], qt, kc, vc, lengths, THETA)
    cached.check(got, qt, kc, vc, lengths, THETA)


def test_replayed_steps_are_the_eager_ones():
    hidden, lengths = 256, [60, 5, 17]
    layers = [Layer(hidden, 4, 2, 8, 2, 128, lengths, 1200) for _ in range(2)]
    for one in layers:
        one.prompt(rnd(sum(lengths), hidden, seed=12), lengths)
    x = rnd(len(lengths), hidden, seed=13)
    eager = []
    for _ in range(5):
        eager.append(layers[0].token(eager[-1] if eager else x)[-1])
    stream, held = torch.cuda.Stream(), x.clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        held.copy_(layers[1].token(held)[-1])
        assert torch.equal(held, eager[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held.copy_(layers[1].token(held)[-1])
        for want in eager[1:]:
            graph.replay()
            assert torch.equal(held, want)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(layers[0].lengths, layers[1].lengths)
    for one, other in ((layers[0].kc, layers[1].kc), (layers[0].vc, layers[1].vc)):
        assert torch.equal(one.view(torch.int16), other.view(torch.int16))
    ops.device_status()


@pytest.mark.parametrize("room", [400, 1500, 17000])
def test_token_steps_hold_the_bound_of_two_part_products(room):
    """The cache attention of a layer's steps, as narrow as its arithmetic allows:
    eagerly, then from a replayed graph whose lengths have grown."""
    hidden, lengths = 256, [130, 0, 33, 300, 1]
    layer = Layer(hidden, 4, 2, 8, 2, 128, lengths, room)
    layer.prompt(rnd(sum(lengths), hidden, seed=20), lengths)
    x, stream = rnd(len(lengths), hidden, seed=21), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _, fused, o, *_ = layer.token(x)
        now = [n + 1 for n in lengths]
        assert _attention.excess(o, layer.split(fused)[0], layer.kc, layer.vc, now, THETA) <= 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, fused, o, *_ = layer.token(x)
        for step in range(3):
            x.copy_(rnd(len(lengths), hidden, seed=22 + step))
            graph.replay()
            now = [n + 1 for n in now]
            assert layer.lengths.tolist() == now
            assert _attention.excess(o, layer.split(fused)[0], layer.kc, layer.vc, now, THETA) <= 0
    torch.cuda.current_stream().wait_stream(stream)
    ops.device_status()
