"""Codes of a 4-bit cache next to half-way between two of them: those of fp32 arithmetic, whose differences and quotients are rounded."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import angles_of, codes_of, int32, quantised

pytestmark = pytest.mark.gpu


def in_32_bits(x):
    """codes [..., 128] and scales of finite fp16 values as fp32 arithmetic gives them, on the CPU: every difference and quotient rounded once, the code half to even"""
    g = x.cpu().numpy().astype(np.float32).reshape(x.shape[:-1] + (4, 32))
    low, high = g.min(-1), g.max(-1)
    scale = ((high - low) / np.float32(15)).astype(np.float16)
    step = scale.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(step > 0, np.minimum(np.rint((g - low[..., None]) / step), 15), 0)
    scales = np.stack((scale, low.astype(np.float16)), -1)
    return torch.from_numpy(n.astype(np.int64)).flatten(-2).cuda(), torch.from_numpy(scales).cuda()


def compare(part, codes, scales):
    n, s = in_32_bits(part)
    assert torch.equal(codes_of(codes)[:, :, 0], n) and torch.equal(scales[:, :, 0], s)
    return (n != quantised(part)[0]).sum().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_symmetric_groups_with_tiny_values(dtype):
    """A minimum of minus the maximum puts 0 half-way between codes 7 and 8: tiny values of both signs, whose differences round to half-way, and others that do not."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, hkv = 60, 2
    x = torch.randint(-6, 7, (tokens, 3 * hkv, 4, 32), generator=g, device="cuda") * 2.0**-24
    x[10:20] = torch.randn(10, 3 * hkv, 4, 32, generator=g, device="cuda") * 1e-4
    x[20:30] = torch.randn(10, 3 * hkv, 4, 32, generator=g, device="cuda") * 1e-2
    most = torch.tensor([15.0, 1.0, 2047.0, 3.3, 0.11, 60000.0, 7.5, 480.0, 1e-3, 30.0], device="cuda")[torch.arange(tokens, device="cuda") % 10]
    x[..., 3], x[..., 20] = -most[:, None, None], most[:, None, None]
    x = x.half().to(dtype).flatten(1)
    cache = ops.kv4_cache(tokens, 1, hkv)
    out = ops.qkv_append(x, int32([0] * tokens), angles_of(1), cache, hkv, hkv)
    assert torch.equal(out, x.half())
    k, v = (t.unflatten(1, (hkv, 128)) for t in out[:, hkv * 128:].chunk(2, dim=1))
    apart = compare(k, cache[0], cache[1]) + compare(v, cache[2], cache[3])
    assert apart > 100                                         # where 64 bits would have the code next to it
    ops.device_status()


@pytest.mark.parametrize("hkv,tokens", [(8, 3), (32, 70), (5, 2000)])
def test_such_groups_behind_the_transform(hkv, tokens):
    """Whole numbers of up to 15 as the transform's result, exactly (x = H y, at most 1920), and angles that shrink all but two of a group's: few tokens, and as many as take the
    transform on the tensor core."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(tokens)
    y = torch.randint(-8, 9, (tokens, 3 * hkv, 128), generator=g, device="cuda").double()
    y[..., 4::32], y[..., 9::32] = -15, 15
    h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for _ in range(7):
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    x = (y @ h).half()
    assert torch.equal(x.double(), y @ h)
    places = 3
    angles = torch.zeros(places, 64, 2, device="cuda")
    angles[..., 0] = torch.tensor([2.0**-24, -(2.0**-24), 1e-5], device="cuda")[:, None] * (1 + torch.arange(64, device="cuda") % 5)
    angles[:, 4::32, 0] = angles[:, 9::32, 0] = 1
    cache = ops.kv4_cache(tokens, places, hkv)
    pos = torch.arange(tokens, device="cuda").int() % places
    out = ops.qkv_append(x.flatten(1), pos, angles, cache, hkv, hkv, scale=128**-0.5, transform=True)
    k = out.unflatten(1, (-1, 128))[:, hkv:2 * hkv]
    turned = y[:, hkv:2 * hkv] * torch.cat((angles[..., 0], angles[..., 0]), -1)[pos.long()][:, None]
    assert torch.equal(k, turned.float().half())
    here = torch.arange(tokens, device="cuda")
    assert compare(k, cache[0][here, :, pos.long()][:, :, None], cache[1][here, :, pos.long()][:, :, None]) > 10
    ops.device_status()


@pytest.mark.parametrize("spread,offset", [(1.0, 0.0), (1e-6, 0.0), (3000.0, 0.0), (0.01, 500.0), (1.0, -1e-3)])
def test_values_are_rounded_once(spread, offset):
    """What a cache's codes stand for, to the bit: minimum + code * scale is exact in 64 bits (fp16's exponents span 40, a product has 15 bits), and rounded to fp16 directly."""
    from rptc_b200 import ops
    from test_gpu_kv4 import decoded, random_cache
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = random_cache(g, 2, 500, 3, spread, offset)
    for i, t in zip((0, 2), ops.kv4_values(cache, int32([500, 333]))):
        want = decoded(cache[i], cache[i + 1]).transpose(1, 2).cpu().numpy().astype(np.float16)
        got = t.cpu().numpy()
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1, :333], want[1, :333])
    ops.device_status()
