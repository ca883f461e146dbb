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
    assert "too many rows" in refused(*call(rows=1 << 31), status=_abi.UNSUPPORTED)
    assert getattr(_abi.lib(), "ennx_b200_gqa_attention_packed")(*call(rows=0)[1:]) == _abi.OK
