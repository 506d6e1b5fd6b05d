"""A decode step whose queries leave fp16 once they are rotated: the Hadamard matrix adds up to sqrt(d) of a channel's size together.  Tolerances are
those of the operators' other tests."""
import pytest
import torch

from test_gpu_cache_i4 import check_decode, decode_case, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "ctypes"])
def ops(request):
    if request.param == "ctypes":
        from flh_amd import _ops
        return _ops
    import flh_amd
    return flh_amd._CUDA


@pytest.mark.parametrize("B,Hq,Hkv,d,n", [(1, 8, 2, 128, 5), (2, 32, 8, 64, 300), (3, 40, 2, 128, 700)])
@pytest.mark.parametrize("size", [6000.0, 65504.0])
def test_rotated_queries_beyond_fp16(ops, B, Hq, Hkv, d, n, size):
    case = decode_case(torch.Generator().manual_seed(n), B, Hq, Hkv, d, n + 1, [n - b for b in range(B)])
    q, cos, sin = case[0], case[3], case[4]
    q[:, 1::3] = size                                                  # (the heads between them are ordinary ones)
    q[0, 0, ::2], q[0, 0, 1::2] = size, -size
    cos[0], sin[0] = 1.0, 0.0
    rotated = turned(q, cos, sin, torch.float64)
    assert rotated[0, :2].abs().amax(-1).min() > 65504 or (size < 8000 and d == 64)
    check_decode(ops, case, scale=1e-6)
    check_decode(ops, case, scale=1e-3)


def test_queries_that_are_not_finite_spoil_themselves(ops):
    case = decode_case(torch.Generator().manual_seed(1), 1, 16, 1, 128, 200, [150])
    q = case[0]
    q[0, 3], q[0, 5, 7], q[0, 9, 1] = 20000.0, float("inf"), float("nan")
    out = ops.decode_attention_rope_i4(*(t.cuda() for t in case[:6]), *(t.cuda() for t in case[6]), scale=1e-5).cpu()
    nan = torch.isnan(out[0])
    assert nan[5].all() and nan[9].all() and not nan[[h for h in range(16) if h not in (5, 9)]].any()
