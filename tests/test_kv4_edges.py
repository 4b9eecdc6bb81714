"""The 4-bit key/value cache's oracle at the ends of its types, without a GPU."""
import pytest
import torch

from oracle import kv4 as okv4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_finite_groups_stay_finite_at_the_end_of_the_type(dtype):
    """Groups that reach the largest number, from minima of every size: read back finite and within half a step."""
    top = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(0)
    x = torch.rand(400, 64, generator=gen, dtype=torch.float64)
    low = torch.linspace(-1.0 if dtype == torch.float16 else 0.0, 0.999, 400, dtype=torch.float64)[:, None]
    x = ((low + (1 - low) * x) * top).to(dtype)
    x[:, 0], x[:, 1] = (low[:, 0] * top).to(dtype), top
    n, s, m = okv4.quantise(x)
    v, back = okv4.values(x)
    assert s.isfinite().all() and back.isfinite().all() and int(n.max()) == 15
    # Half a step, fp32's rounding of the difference, and for the read-back its own rounding.
    room = okv4.spread(s) * 0.5 * (1 + 2.0 ** -20)
    assert ((v - x.double()).abs() <= room).all()
    assert ((back.double() - x.double()).abs() <= room + x.double().abs() * torch.finfo(dtype).eps).all()
    # Away from the end the step is the smallest one that holds the range.
    n, s, m = okv4.quantise((x.double() / 4).to(dtype))
    y = (x.double() / 4).to(dtype)
    assert ((y.amax(-1).double() - y.amin(-1).double()) / 15 <= s[:, 0].double() * (1 + 2.0 ** -22)).all()
