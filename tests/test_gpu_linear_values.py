"""GPU: values at the ends of their types in compressed weights (nncf_amd.linear), against the plain product in 64 bits with the
bounds of tests/linear_utils.py."""
import pytest
import torch

from tests.linear_utils import assert_within, make_weight, plain

pytestmark = pytest.mark.gpu


def _rows(m, k, dtype, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _nibbles(values):
    return (values[..., 0::2] | (values[..., 1::2] << 4)).reshape(-1, 1).contiguous()


@pytest.mark.parametrize("m", [1, 5, 16, 33, 64, 130, 300])
@pytest.mark.parametrize("mode,gs,n,k,dtype", [("int4_sym", 64, 64, 320, torch.bfloat16), ("int4_sym", 32, 48, 352, torch.bfloat16),
                                               ("int4_sym", 32, 33, 32, torch.bfloat16), ("int4_asym", 64, 80, 448, torch.bfloat16),
                                               ("int4_asym", 32, 16, 96, torch.bfloat16), ("int4_sym", 64, 130, 4160, torch.bfloat16),
                                               ("mxfp4", 32, 64, 416, torch.float16), ("mxfp4", 32, 16, 4128, torch.float16)])
def test_a_large_scale_meets_its_own_codes_only(mode, gs, n, k, dtype, m):
    """The last group's scale is so large that codes of other groups would leave fp16 under it, while its own do not: the weight is
    finite, and what lies behind the end of k must not bring an infinity in (times x's zeros it would be NaN)."""
    from nncf_amd.linear import compressed_linear
    packed, dec = make_weight(mode, gs, (n, k), dtype, seed=k)
    codes = torch.randint(0, 16, (n, k), dtype=torch.uint8, generator=torch.Generator().manual_seed(m)).cuda()
    last = codes[:, k - gs:]
    last.remainder_(2)  # mxfp4: 0 and 0.5
    if mode == "mxfp4":
        dec._scale[:, -1] = 127 + 15
        codes[:, : min(32, k - gs)] = 7  # 6
    else:
        if mode == "int4_sym":
            last.add_(7)  # -1 and 0
        else:
            dec._zero_point.zero_()  # 0 and 1
        dec._scale[:, -1] = 16000.0
        codes[:, : min(32, k - gs)] = 15
        codes[:, 0] = 0 if mode == "int4_sym" and k > gs else codes[:, 0]
    packed.copy_(_nibbles(codes))
    w = dec(packed)
    assert bool(torch.isfinite(w).all())
    x = _rows(m, k, dtype, m) * (2.0 ** -10)
    y, by = plain(x, w)
    assert_within(compressed_linear(x, packed, dec), y, by)
