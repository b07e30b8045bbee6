"""The codes of the 8-bit norm are those of its definition, e4m3(s w / (max|s w| / 448)), rounded operation by operation, and so
the same from whatever kernel a layout and a size lead to: rstd, whose last bit hangs on the order of a sum, is in the scale alone."""
import pytest
import torch

import _network_ops as ref
from spherical_distortion import functional as F

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn
EPS = 1e-6


def normal(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale


def codes_of(s, w):
    """Of rows (n, C)."""
    p = s.float() * w.float() if w is not None else s.float()
    return (p * (p.abs().amax(1, keepdim=True).reciprocal() * 448.0)).to(E4)


def layouts(rows):
    """{name: (tensor, dim, rows back)} of the same rows in every layout that has a kernel of its own."""
    n, c = rows.shape

    def planes(count):
        x = rows[:count].t().contiguous()
        return x.view(1, c, count), 1, lambda t: t.view(c, -1).t()
    one_off = torch.cat([rows.new_zeros(1), rows.reshape(-1)])[1:].view(n, c)
    wider = torch.cat([rows, rows.new_zeros(n, 1)], 1)[:, :c]
    same = lambda t: t  # noqa: E731
    # (128 pixels start on 16-byte boundaries, 1001 and 49 do not, and the last are too few for shifted runs)
    return {"rows": (rows, -1, same), "one off": (one_off, -1, same), "odd strides": (wider, -1, same), "aligned planes": planes(128),
            "odd planes": planes(1001), "small planes": planes(49)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c", [24, 40, 96, 300, 500, 1032, 5000, 20000])
def test_codes_do_not_depend_on_the_kernel(c, dtype):
    rows, w = normal((1001, c), c, 1.5).to(dtype), normal((c,), c + 1) * 0.2 + 1
    add = normal((1001, c), c + 2).to(dtype)
    for weight in (w, w.to(dtype), None):
        for residual in (False, True):
            s = (rows.float() + add.float()).to(dtype) if residual else rows
            want = codes_of(s, weight)
            for name, (x, dim, back) in layouts(rows).items():
                r = layouts(add)[name][0] if residual else None
                if r is not None and not r.is_contiguous():
                    r = r.contiguous()
                q, scale, *_ = F.rms_norm_quantized(x, weight, r, EPS, dim)
                got = back(q.float())
                assert torch.equal(got, want[:len(got)].float()), (name, residual, (got != want[:len(got)].float()).sum().item())


def test_codes_of_rows_without_a_scale():
    """Zeros, values too small for a scale, infinities and NaN, from each kernel."""
    for c in (40, 300, 5000, 20000):
        rows = normal((1001, c), 7)
        rows[0], rows[1], rows[2, 3], rows[3, 5] = 0, 1e-36, float("inf"), float("nan")
        for name, (x, dim, back) in layouts(rows).items():
            q, scale = F.rms_norm_quantized(x, None, None, EPS, dim)
            got, scale = back(q.float()), scale.reshape(-1)
            assert not got[:2].any() and not scale[:2].any(), name
            assert torch.isnan(got[2, 3]) and torch.isnan(got[3]).all() and torch.isnan(scale[2:4]).all(), name
            assert torch.isfinite(got[4:]).all() and torch.isfinite(scale[4:]).all(), name


@pytest.mark.parametrize("seed", range(4))
def test_a_code_differs_from_64_bits_only_at_a_border(seed):
    """Three roundings (product, reciprocal, its multiple) and the last product may carry a value over a border of two codes that
    is nearer than 4.1 of them; nowhere else, and never further than to the next code."""
    s, w = normal((4000, 96), seed, 1.5).bfloat16(), normal((96,), seed + 9) * 0.2 + 1
    q, _ = F.rms_norm_quantized(s, w, None, EPS, -1)
    exact = s.double() * w.double()
    exact = exact / exact.abs().amax(1, keepdim=True) * 448
    low, high = (exact * (1 - 4.1 * ref.U)).float().to(E4).float(), (exact * (1 + 4.1 * ref.U)).float().to(E4).float()
    got = q.float()
    assert ((got == low) | (got == high)).all()
