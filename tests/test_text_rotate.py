"""text_decoder.rotate on the CPU against complex numbers in float64: two products and a sum in float32, each
within half a step, 2^-24, of values that |a| + |b| bounds."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd.text_decoder import rotate


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,dim", [(0, 2, 8), (1, 1, 2), (7, 3, 64), (33, 2, 128)])
def test_rotate(tokens, heads, dim, dtype):
    g = torch.Generator().manual_seed(dim)
    x = torch.randn((tokens, heads, dim), generator=g).to(dtype)
    angle = torch.rand((tokens, dim // 2), generator=g, dtype=torch.float64) * 100
    cos, sin = angle.cos().float(), angle.sin().float()
    got = rotate(x, cos, sin)
    assert got.dtype == torch.float32 and got.shape == x.shape
    a, b = x.double().chunk(2, -1)
    z = torch.complex(a, b) * torch.complex(cos.double(), sin.double())[:, None]
    size = torch.cat([a.abs() + b.abs()] * 2, -1)
    assert ((got.double() - torch.cat([z.real, z.imag], -1)).abs() <= 2.0 ** -23 * size).all()
