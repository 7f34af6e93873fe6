"""The 8-bit cache's reference against torch's own conversions and against differences that its definition bounds (CPU)."""
import pytest
import torch

import kv8_ref as R

CODES = [torch.int8, torch.float8_e4m3fn]


def test_e4m3_grid_is_torch_float8():
    x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(torch.half)
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert torch.equal(R.codes_of(x, 1.0, torch.float8_e4m3fn), x.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("dtype", CODES)
def test_scale_is_the_smallest_power_that_holds_the_block(dtype):
    for top in (0.0, 2.0 ** -24, 1e-6, 0.03, 1.0, 126.9375, 127.0, 127.0625, 448.0, 448.25, 4096.0, 65504.0):
        s = R.scale_of(torch.tensor([top, -top / 3]).half(), dtype)
        v = float(torch.tensor(top).half())
        assert v <= R.MOST[dtype] * s and (s == 2.0 ** -24 or v > R.MOST[dtype] * s / 2)
        assert abs(float(R.codes_of(torch.tensor([v]), s, dtype)[0]) * s) <= 65504


@pytest.mark.parametrize("dtype", CODES)
def test_block_that_grows_stays_within_one_step(dtype):
    """Sixteen tokens one by one, each larger than the ones before: int8 within the last scale, e4m3 within half a step of
    the value or of the subnormals at the last scale, twice."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(16, 1, 64, generator=g) * (1.6 ** torch.arange(16.0))[:, None, None]).half()
    kc, ks = torch.zeros(1, 1, 16, 64, dtype=dtype), torch.zeros(1, 1, 1)
    vc, vs = kc.clone(), ks.clone()
    bt = torch.zeros(1, dtype=torch.int32)
    for t in range(16):
        _, (kc, vc, ks, vs) = R.append(torch.cat([x[t], x[t], x[t]], 1), None, None, t, bt, kc, vc, ks, vs, 1)
    s, got = float(ks), R.values(kc, ks)[0, 0]
    err, want = (got - x[:, 0].double()).abs(), x[:, 0].double().abs()
    assert torch.equal(kc, vc) and s > 64 * R.scale_of(x[:1], dtype)
    step = s if dtype == torch.int8 else 2.0 ** -4 * want + 2 * 2.0 ** -10 * s
    assert bool((err <= step).all())
