"""Refusals of the serving operators that the host makes before any device work."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ennx_b200 import _abi, ops  # noqa: E402

P = ctypes.c_void_p
BF16 = torch.bfloat16


def refused(name, *args, status=_abi.INVALID_ARGUMENT):
    st = getattr(_abi.lib(), name)(*args)
    assert st == status, (st, _abi.lib().ennx_b200_last_error())
    return _abi.lib().ennx_b200_last_error().decode()


def test_packed_attention_refuses_on_the_host():
    q = torch.zeros(4, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gqa_attention_packed(q, q, q, torch.zeros(2, dtype=torch.int32))
    a = P(256)

    def call(q=a, ldq=512, k=a, ldk=256, v=a, ldv=256, o=a, ldo=512, cu=a, n=1, rows=8, hq=4, hkv=2, theta=0.0):
        return ("ennx_b200_gqa_attention_packed", q, ldq, k, ldk, v, ldv, o, ldo, cu, n, rows, hq, hkv, theta, None)

    assert "no sequences" in refused(*call(n=0))
    assert "no sequences" in refused(*call(cu=None))
    assert "multiple of Hkv" in refused(*call(hq=3))
    assert "multiple of Hkv" in refused(*call(rows=-1))
    assert "null" in refused(*call(o=None))
    assert "shorter" in refused(*call(ldq=504))
    assert "aligned" in refused(*call(ldk=260))
    assert "aligned" in refused(*call(v=P(264 + 2)))
    assert "rope_theta" in refused(*call(theta=float("nan")))
    assert "cannot be shared" in refused(*call(ldq=512, theta=1e6))
    assert "too many rows" in refused(*call(rows=1 << 31), status=_abi.UNSUPPORTED)
    assert getattr(_abi.lib(), "ennx_b200_gqa_attention_packed")(*call(rows=0)[1:]) == _abi.OK


def test_decode_attention_refuses_on_the_host():
    def call(theta=0.0, workspace=P(256), size=1 << 30, **over):
        f = dict(q=256, ld_q=512, k=256, ld_k=256, v=256, ld_v=256, k_cache=256, k_seq=8192, k_token=256, k_head=128,
                 v_cache=256, v_seq=8192, v_token=256, v_head=128, lengths=256, o=256, ld_o=512, batch=2, room=1 << 20,
                 hq=4, hkv=2)
        f.update(over)
        return ("ennx_b200_gqa_attention_decode", ctypes.byref(_abi.DecodeAttention(**f)), theta, workspace, size, None)

    assert "null parameters" in refused("ennx_b200_gqa_attention_decode", None, 0.0, None, 0, None)
    assert "room" in refused(*call(room=0))
    assert "multiple of Hkv" in refused(*call(hq=5))
    assert "rope_theta" in refused(*call(theta=-1.0))
    assert "null argument" in refused(*call(lengths=0))
    assert "come together" in refused(*call(v=0))
    assert "shorter" in refused(*call(ld_q=504))
    assert "shorter" in refused(*call(ld_k=128))
    assert "negative" in refused(*call(k_seq=-8192))
    assert "multiple of 8" in refused(*call(v_token=260))
    assert "aligned" in refused(*call(k_cache=260))
    assert "must be apart" in refused(*call())
    assert "strides of 0" in refused(*call(k_seq=0))
    many = dict(batch=1 << 20, hq=1 << 8, hkv=1 << 8, room=(1 << 31) - 1, k=0, v=0, ld_q=1 << 15, ld_o=1 << 15)
    assert "too many" in refused(*call(**many), status=_abi.UNSUPPORTED)
    assert "strides of 0" in refused(*call(v_head=0))
    assert "strides of 0" in refused(*call(v_token=0))
    assert "workspace" in refused(*call(k=0, v=0, k_seq=0, workspace=None))  # caches that are only read may share
    apart = dict(v_cache=1 << 40)
    assert "workspace" in refused(*call(workspace=None, **apart))
    assert "workspace" in refused(*call(size=1000, **apart))
    assert "workspace" in refused(*call(workspace=P(260), **apart))
    assert getattr(_abi.lib(), "ennx_b200_gqa_attention_decode")(*call(batch=0)[1:]) == _abi.OK
    q = torch.zeros(2, 4, 128, dtype=BF16)
    c = torch.zeros(2, 8, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gqa_attention_decode(q, c, c, torch.zeros(2, dtype=torch.int32))


def test_moe_layer_decode_refuses_on_the_host():
    a = P(256)

    def call(x=a, wr=a, wgu=a, wd=a, t=2, h=256, e=8, k=2, i=128, y=a, ws=a, size=1 << 30):
        return ("ennx_b200_moe_layer_decode", x, wr, wgu, wd, t, h, e, k, i, None, y, None, None, ws, size, None)

    assert "negative" in refused(*call(t=-1))
    assert "top_k" in refused(*call(k=9))
    assert "top_k" in refused(*call(e=1))
    assert "at most 64 tokens" in refused(*call(t=65), status=_abi.UNSUPPORTED)
    assert "256 experts" in refused(*call(e=257), status=_abi.UNSUPPORTED)
    assert "multiple of 64" in refused(*call(h=96), status=_abi.UNSUPPORTED)
    assert "multiple of 64" in refused(*call(i=192), status=_abi.UNSUPPORTED)
    assert "null" in refused(*call(wd=None))
    assert "aligned" in refused(*call(x=P(258)))
    assert "workspace" in refused(*call(size=100))
    assert "workspace" in refused(*call(ws=P(8)))
    assert _abi.lib().ennx_b200_moe_layer_decode(*call(t=0)[1:]) == _abi.OK
    x = torch.zeros(2, 256, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_layer_decode(x, torch.zeros(8, 256, dtype=BF16), torch.zeros(8, 256, 256, dtype=BF16),
                             torch.zeros(8, 256, 128, dtype=BF16), 2)


def test_packed_linear_decode_refuses_on_the_host():
    a, seed = P(256), _abi.PerturbSeed(0, 0, 0)
    lin = _abi.PackedLinear(0, 0, 0, 64, 8, 4, 32, 0, 0, 0)

    def call(x=a, t=2, w=a, sc=a, bi=a, d=lin, out=a):
        return ("ennx_b200_packed_linear_decode", x, t, w, sc, bi, None if d is None else ctypes.byref(d), seed, out,
                None)

    assert "descriptor is null" in refused(*call(d=None))
    assert "bits must be 4 or 8" in refused(*call(d=_abi.PackedLinear(0, 0, 0, 64, 8, 3, 32, 0, 0, 0)))
    assert "must be positive" in refused(*call(d=_abi.PackedLinear(0, 0, 0, 64, 8, 4, 0, 0, 0, 0)))
    assert "negative" in refused(*call(t=-1))
    assert "at most 16 tokens" in refused(*call(t=17), status=_abi.UNSUPPORTED)
    assert "2^31" in refused(*call(d=_abi.PackedLinear(0, 0, 0, 1 << 31, 8, 4, 32, 0, 0, 0)), status=_abi.UNSUPPORTED)
    assert "null" in refused(*call(bi=None))
    assert "misaligned" in refused(*call(sc=P(258)))
    assert "misaligned" in refused(*call(x=P(257)))
    assert _abi.lib().ennx_b200_packed_linear_decode(*call(t=0)[1:]) == _abi.OK
    with pytest.raises(ValueError, match="CUDA"):
        ops.packed_linear_decode(torch.zeros(2, 64, dtype=BF16), torch.zeros(256, dtype=torch.uint8), torch.zeros(16),
                                 torch.zeros(16), lin)


def test_packed_attention_refuses_memory_that_is_shared():
    def call(q=1 << 40, k=(1 << 40) + 1024, v=(1 << 40) + 1536, o=1 << 41, cu=1 << 42, ld=1024, ldo=512, theta=0.0, rows=8):
        return ("ennx_b200_gqa_attention_packed", P(q), ld, P(k), ld, P(v), ld, P(o), ldo, P(cu), 1, rows, 4, 2, theta, None)

    for over in (dict(o=1 << 40, ldo=1024), dict(o=(1 << 40) + 512), dict(o=(1 << 40) + 1536, ldo=1024),
                 dict(o=(1 << 40) - 7 * 1024, ldo=512), dict(cu=(1 << 41) + 1020), dict(o=(1 << 40) + 1024, ldo=1024),
                 dict(o=(1 << 40) + 7 * 2048 + 2032)):
        assert "must not overlap" in refused(*call(**over))
    for over in (dict(k=(1 << 40) + 1008), dict(v=(1 << 40) + 2048), dict(v=(1 << 40) + 1520), dict(k=1 << 40),
                 dict(cu=(1 << 40) + 2044)):
        assert "in place" in refused(*call(theta=1e6, **over))


def test_decode_attention_refuses_memory_that_is_shared():
    base = 1 << 40

    def call(**over):
        f = dict(q=base, ld_q=1024, k=base + 1024, ld_k=1024, v=base + 1536, ld_v=1024, k_cache=1 << 41, k_seq=8192,
                 k_token=256, k_head=128, v_cache=1 << 42, v_seq=8192, v_token=256, v_head=128, lengths=1 << 43, o=1 << 44,
                 ld_o=512, batch=4, room=32, hq=4, hkv=2)
        f.update(over)
        return ("ennx_b200_gqa_attention_decode", ctypes.byref(_abi.DecodeAttention(**f)), 0.0, None, 0, None)

    for over in (dict(o=base + 16, ld_o=1024), dict(o=base), dict(o=base - 2048, ld_o=1024), dict(o=base + 512)):
        assert "q itself" in refused(*call(**over))
    reads = dict(k=0, v=0)
    for over in (dict(o=base + 1024, ld_o=1024), dict(o=(1 << 41) + 8192), dict(o=(1 << 42) + 4 * 8192 * 2 - 16),
                 dict(o=(1 << 43) - 1024 * 3 - 1008), dict(o=(1 << 41) + 8192, **reads)):
        assert "o must not overlap" in refused(*call(**over))
    for over in (dict(k_head=120), dict(k_token=64, k_head=32 * 64, k_seq=2 * 32 * 64), dict(v_seq=8192 - 128)):
        assert "rows of a cache" in refused(*call(**over))
    for over in (dict(v_cache=(1 << 41) + 256), dict(v_cache=(1 << 41) + 8192 * 2 - 16)):
        assert "must be apart" in refused(*call(**over))
    for over in (dict(k_cache=base + 2048), dict(v_cache=base + 1024), dict(k_cache=(1 << 43) - 8192)):
        assert "caches that take" in refused(*call(**over))


def test_moe_layer_decode_refuses_memory_that_is_shared():
    far = [1 << (40 + i) for i in range(9)]

    def call(x=far[0], wr=far[1], wgu=far[2], wd=far[3], res=far[4], y=far[5], index=far[6], gate=far[7], ws=far[8]):
        p = [P(a) for a in (x, wr, wgu, wd)]
        return ("ennx_b200_moe_layer_decode", *p, 3, 256, 8, 2, 128, P(res), P(y), P(index), P(gate), P(ws), 1 << 20, None)

    size = 3 * 256 * 2
    for over in (dict(y=far[0]), dict(y=far[0] + size - 2), dict(y=far[1] + 8 * 512 - 2), dict(y=far[2] + 8 * 256 * 512 - 2),
                 dict(y=far[3] + 8 * 256 * 256 - 2), dict(y=far[4] + 2), dict(y=far[4] - size + 2), dict(index=far[0]),
                 dict(gate=far[4] + 8), dict(ws=far[3] + 16), dict(ws=far[0] - 16)):
        assert "must not overlap x" in refused(*call(**over))
    for over in (dict(index=far[5]), dict(gate=far[6] + 20), dict(ws=far[7] - 16), dict(y=far[8])):
        assert "workspace must not overlap" in refused(*call(**over))


def test_packed_linear_decode_refuses_memory_that_is_shared():
    far = [1 << (40 + i) for i in range(5)]
    lin = _abi.PackedLinear(64, 16, 32, 100, 8, 4, 32, 0, 0, 0)  # codes 8 x 50 bytes, scales and biases 8 x 4 floats

    def call(x=far[0], w=far[1], sc=far[2], bi=far[3], out=far[4]):
        return ("ennx_b200_packed_linear_decode", P(x), 3, P(w), P(sc), P(bi), ctypes.byref(lin),
                _abi.PerturbSeed(0, 0, 0), P(out), None)

    size = 3 * 8 * 2
    for out in (far[0], far[0] + 3 * 200 - 2, far[0] - size + 2, far[1] + 64 + 398, far[1] + 64 - size + 2,
                far[2] + 64 + 126, far[2] + 64 - size + 2, far[3] + 128 + 126, far[3] + 128 - size + 2):
        assert "must not overlap" in refused(*call(out=out))


def test_heads_whose_columns_pass_32_bits_are_refused():
    heads, far = 1 << 24, [P(1 << (40 + i)) for i in range(7)]
    assert "too many" in refused("ennx_b200_gqa_attention_packed", far[0], heads * 128, far[1], 128, far[2], 128, far[3],
                                 heads * 128, far[4], 1, 1, heads, 1, 0.0, None, status=_abi.UNSUPPORTED)
    p = _abi.DecodeAttention(q=1 << 40, ld_q=heads * 128, k=1 << 41, ld_k=heads * 128, v=1 << 42, ld_v=heads * 128,
                             k_cache=1 << 43, k_seq=0, k_token=0, k_head=128, v_cache=1 << 44, v_seq=0, v_token=0,
                             v_head=128, lengths=1 << 45, o=1 << 46, ld_o=heads * 128, batch=1, room=1, hq=heads, hkv=heads)
    assert "too many" in refused("ennx_b200_gqa_attention_decode", ctypes.byref(p), 0.0, None, 0, None,
                                 status=_abi.UNSUPPORTED)
