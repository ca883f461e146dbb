"""Few-token packed products on the GPU against their definition in 64 bits,
the codes taken from the oracle-checked dequantisation.

Tolerance: codes and activations are exact in bf16 and so are their products in
fp32; sums are fp32.  A chain has at most K additions, each off by at most
2^-23 of a running magnitude below A = sum |code x| |scale| + |bias x|: with the
256 columns of a chain joined as a tree, 2^-23 * 280 * A <= 2^-14 A bounds it for
every width here.  The result is rounded to bf16 once (2^-8 relative)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ennx_b200 import _abi, ops  # noqa: E402


def make(inp, out, bits, group, seed, offsets=(0, 0, 0), whole=0, threshold=0, element=0):
    rng = np.random.default_rng(seed)
    row_bytes, groups = (inp * bits + 7) // 8, -(-inp // group)
    w = rng.integers(0, 256, offsets[0] + out * row_bytes, dtype=np.uint8)
    sc = rng.uniform(0.5, 1.5, offsets[1] + out * groups).astype(np.float32) * 3.0 / ((1 << bits) * inp ** 0.5)
    bi = -rng.uniform(0.4, 0.6, offsets[2] + out * groups).astype(np.float32) * 3.0 / inp ** 0.5
    lin = _abi.PackedLinear(*offsets, inp, out, bits, group, element, whole, threshold)
    return [torch.from_numpy(a).cuda() for a in (w, sc, bi)] + [lin]


def x_of(tokens, inp, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, inp, generator=g, device="cuda").to(torch.bfloat16)


def check(got, x, w, sc, bi, lin, seed=(0, 0, 0)):
    inp, out, group = lin.input_width, lin.output_width, lin.group_size
    groups = -(-inp // group)
    # the code itself: dequantise with scale 1 and bias 0
    codes = ops.packed_dequantize(w, torch.ones_like(sc), torch.zeros_like(bi), lin, seed, dtype=torch.float32).double()
    column = torch.arange(inp, device="cuda") // group
    s = sc[lin.scale_offset:lin.scale_offset + out * groups].view(out, groups).double()[:, column]
    b = bi[lin.bias_offset:lin.bias_offset + out * groups].view(out, groups).double()[:, column]
    ref = x.double() @ (codes * s + b).T
    size = x.double().abs() @ (codes * s.abs() + b.abs()).T
    err = (got.double() - ref).abs() - (1.001 * 2.0 ** -8 * ref.abs() + 2.0 ** -14 * size)
    assert err.max() <= 0, float(err.max())


SHAPES = [
    (4096, 40, 128), (8192, 50, 256), (2048, 333, 512), (6144, 21, 64), (4096, 2500, 32), (512, 700, 128),
    (2048, 512, 64), (256, 48, 32), (64, 16, 64), (32, 1, 32), (1, 1, 1), (7, 3, 4), (200, 17, 48), (37, 9, 8), (16, 33, 16),
    (512, 100, 128), (1024, 31, 256), (2048, 40, 2048), (96, 300, 16), (4096, 64, 64), (4160, 24, 32), (8200, 19, 64),
    (2011, 50, 64), (255, 65, 32), (1000, 20, 1000), (2080, 16, 96), (130, 130, 160), (2304, 8, 2000),
]


@pytest.mark.parametrize("inp,out,group", SHAPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens", [1, 3, 8, 9, 16])
def test_matches_definition(inp, out, group, bits, tokens):
    w, sc, bi, lin = make(inp, out, bits, group, inp + bits)
    x = x_of(tokens, inp, tokens)
    check(ops.packed_linear_decode(x, w, sc, bi, lin), x, w, sc, bi, lin)


@pytest.mark.parametrize("inp,out,group", [(256, 33, 32), (2048, 64, 64), (201, 40, 32), (37, 9, 8), (96, 20, 16)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("whole,threshold,element", [(0, 0x40000000, 5), (1, 1 << 31, 2 ** 32 - 300), (20, 0, 0), (0, 1, 0),
                                                     (300, 0xFFFFFFFF, 7)])
def test_moved_codes(inp, out, group, bits, whole, threshold, element):
    w, sc, bi, lin = make(inp, out, bits, group, 3, whole=whole, threshold=threshold, element=element)
    x, seed = x_of(5, inp, 4), (0x9E37, 0x51ED27, 1)
    check(ops.packed_linear_decode(x, w, sc, bi, lin, seed), x, w, sc, bi, lin, seed)


@pytest.mark.parametrize("offsets", [(1, 1, 3), (3, 2, 1), (16, 4, 4), (18, 5, 0), (7, 0, 0)])
@pytest.mark.parametrize("inp,group", [(2048, 64), (320, 32), (99, 32)])
@pytest.mark.parametrize("bits", [4, 8])
def test_arena_offsets_of_any_alignment(offsets, inp, group, bits):
    w, sc, bi, lin = make(inp, 70, bits, group, 5, offsets=offsets)
    big = x_of(4, inp + 1, 6).flatten()
    x = big[1:1 + 3 * inp].view(3, inp)  # two-byte aligned only
    check(ops.packed_linear_decode(x, w, sc, bi, lin), x, w, sc, bi, lin)


def test_same_sign_activations():
    # every activation positive: the largest sums the codes can make
    w, sc, bi, lin = make(4096, 32, 8, 64, 8)
    x = x_of(16, 4096, 9).abs() + 1
    check(ops.packed_linear_decode(x, w, sc, bi, lin), x, w, sc, bi, lin)


def test_a_bad_token_or_row_stays_alone():
    w, sc, bi, lin = make(512, 40, 4, 64, 10)
    x = x_of(9, 512, 11)
    clean = ops.packed_linear_decode(x, w, sc, bi, lin)
    x[4, 100] = float("nan")
    sc[3 * 8 + 2] = float("inf")
    y = ops.packed_linear_decode(x, w, sc, bi, lin)
    rows = [r for r in range(40) if r != 3]
    tok = [t for t in range(9) if t != 4]
    assert torch.equal(y[tok][:, rows], clean[tok][:, rows])
    assert y[4].isnan().all() and not y[:, 3].isfinite().any()


def test_graph_out_and_stream():
    w, sc, bi, lin = make(1024, 96, 4, 64, 12)
    x, out = x_of(2, 1024, 13), torch.empty(2, 96, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.packed_linear_decode(x, w, sc, bi, lin, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.packed_linear_decode(x, w, sc, bi, lin, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (14, 15):
        x.copy_(x_of(2, 1024, seed))
        graph.replay()
        check(out, x, w, sc, bi, lin)


def test_no_tokens():
    w, sc, bi, lin = make(64, 8, 4, 32, 16)
    assert ops.packed_linear_decode(x_of(1, 64, 0)[:0], w, sc, bi, lin).shape == (0, 8)


def test_refusals():
    w, sc, bi, lin = make(64, 8, 4, 32, 17)
    x, call = x_of(2, 64, 18), ops.packed_linear_decode
    with pytest.raises(Exception, match="at most 16 tokens"):
        call(x_of(17, 64, 19), w, sc, bi, lin)
    with pytest.raises(ValueError, match="input_width"):
        call(x[:, :32], w, sc, bi, lin)
    with pytest.raises(ValueError, match="exceeds its arenas"):
        call(x, w[:-1], sc, bi, lin)
    with pytest.raises(ValueError, match="exceeds its arenas"):
        call(x, w, sc, bi[:-1], lin)
    with pytest.raises(ValueError, match="uint8"):
        call(x, w.int(), sc, bi, lin)
    with pytest.raises(ValueError, match="bits must be 4 or 8"):
        call(x, w, sc, bi, _abi.PackedLinear(0, 0, 0, 64, 8, 5, 32, 0, 0, 0))
    with pytest.raises(ValueError, match="out must be"):
        call(x, w, sc, bi, lin, out=torch.empty(2, 9, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("inp,group", [(2048, 64), (96, 32), (301, 64)])
def test_rows_of_zero_codes_without_bias_give_zero(inp, group):
    w, sc, bi, lin = make(inp, 48, 4, group, 20)
    w.view(48, -1)[5:40] = 0
    bi.view(48, -1)[5:40] = 0
    y = ops.packed_linear_decode(x_of(11, inp, 21) * 100, w, sc, bi, lin)
    assert (y[:, 5:40] == 0).all() and (y[:, :5] != 0).any()


@pytest.mark.parametrize("bits,inp,group,offset,moved,tokens", [
    (8, (1 << 29) + 1056, 96, 0, False, 1),   # codes copied row by row
    (8, (1 << 29) + 1024, 64, 0, False, 9),   # as boxes, by each warp
    (4, (1 << 30) + 1024, 64, 0, False, 1),   # by one warp, scales too
    (8, (1 << 29) + 1053, 96, 3, False, 1),   # rows at any byte
    (8, (1 << 29) + 1056, 96, 0, True, 1),
    (4, (1 << 30) + 1056, 96, 0, False, 1),
    (4, (1 << 30) + 1050, 96, 5, False, 1),
])
def test_columns_whose_bits_pass_32_bits(bits, inp, group, offset, moved, tokens):
    """Rows of more than 2^32 bits: only the last columns have an activation, the
    first ones hold other codes than the last."""
    rows, tail = 2, 1000
    row_bytes, groups = (inp * bits + 7) // 8, -(-inp // group)
    w = torch.full((offset + rows * row_bytes,), 0x5A, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(30)
    w[offset:].view(rows, row_bytes)[:, -tail * bits // 8:] = torch.randint(0, 256, (rows, tail * bits // 8), device="cuda",
                                                                           generator=g, dtype=torch.uint8)
    sc, bi = torch.full((rows * groups,), 0.5, device="cuda"), torch.zeros(rows * groups, device="cuda")
    lin = _abi.PackedLinear(offset, 0, 0, inp, rows, bits, group, 7, 1, 1 << 31)
    x = torch.zeros(tokens, inp, dtype=torch.bfloat16, device="cuda")
    x[-1, -tail:] = x_of(1, tail, 31)[0]
    seed = (0x9E37, 0x51ED27, int(moved))
    codes = ops.packed_dequantize(w, torch.ones_like(sc), bi, lin, seed, dtype=torch.float32)[:, -tail:].double()
    if not moved:  # the dequantised codes are those of the arena
        end = w[offset:].view(rows, row_bytes)[:, -tail * bits // 8:].long()
        assert torch.equal(codes, (end if bits == 8 else torch.stack([end & 15, end >> 4], 2).flatten(1)).double())
    out = ops.packed_linear_decode(x, w, sc, bi, lin, seed)
    assert (out[:-1] == 0).all()
    got, xt = out[-1].double(), x[-1, -tail:].double()
    ref, size = codes @ xt * 0.5, codes @ xt.abs() * 0.5
    assert ((got - ref).abs() <= 1.001 * 2.0 ** -8 * ref.abs() + 2.0 ** -14 * size).all()


def test_out_that_shares_memory_is_refused():
    w, sc, bi, lin = make(64, 64, 4, 32, 40, offsets=(256, 64, 64))
    x, call = x_of(4, 64, 41), ops.packed_linear_decode
    both = torch.cat([x, x])
    for out in (x, w[256:768].view(torch.bfloat16).view(4, 64), sc[64:192].view(torch.bfloat16).view(4, 64),
                bi[64:192].view(torch.bfloat16).view(4, 64)):
        with pytest.raises(ValueError, match="must not overlap"):
            call(x, w, sc, bi, lin, out=out)
    with pytest.raises(ValueError, match="must not overlap"):
        call(both[:4], w, sc, bi, lin, out=both[3:7])
    assert torch.equal(call(both[:4], w, sc, bi, lin, out=both[4:]), call(x, w, sc, bi, lin))


@pytest.mark.parametrize("bits,group,tokens,moved,skew", [(8, 64, 3, False, 0), (8, 32, 11, False, 0), (8, 64, 16, False, 0),
                                                          (4, 64, 2, False, 0), (4, 32, 16, False, 0), (8, 64, 2, False, 1),
                                                          (8, 64, 4, True, 0), (8, 16, 1, False, 0)])
def test_rows_whose_offsets_pass_32_bits(bits, group, tokens, moved, skew):
    inp, last = 2048, 40
    row_bytes, groups = inp * bits // 8, inp // group
    rows = (1 << 32) // row_bytes + 100
    g = torch.Generator(device="cuda").manual_seed(50)
    w = torch.randint(0, 256, (skew + rows * row_bytes,), generator=g, device="cuda", dtype=torch.uint8)
    sc = torch.rand(rows * groups, generator=g, device="cuda") * 1e-3
    bi = -sc * (1 << (bits - 1))
    x, seed = x_of(tokens, inp, 51), (3, 4, int(moved))
    whole = _abi.PackedLinear(skew, 0, 0, inp, rows, bits, group, 0, 1, 1 << 30)
    got = ops.packed_linear_decode(x, w, sc, bi, whole, seed)
    for first in (0, rows - last):  # rows of the large linear are those of a small one at their place
        part = _abi.PackedLinear(skew + first * row_bytes, first * groups, first * groups, inp, last, bits, group,
                                 first * inp % 2 ** 32, 1, 1 << 30)
        check(got[:, first:first + last], x, w, sc, bi, part, seed)
