"""Appends to a KV cache whose x is written by the call that reads it: cleared, or the result's place, with heads in odd numbers."""
import pytest
import torch

from test_gpu_kv4 import angles_of, codes_of, int32, quantised

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (15, 5), (9, 9), (8, 2)])
@pytest.mark.parametrize("tokens", [1, 6, 700])
@pytest.mark.parametrize("how", ["cleared", "in place"])
def test_x_is_read_before_it_is_written(bits, hq, hkv, tokens, how):
    """Position 0, no transform: what leaves is x * 3, rounded once, to the bit (the product of sixteen bits by two is exact in 32)."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(hq + tokens)
    width = (hq + 2 * hkv) * 128
    x = torch.randn(tokens, width, generator=g, device="cuda").half()
    want = (x.float() * 3).half()
    cache = ops.kv4_cache(tokens, 1, hkv) if bits == 4 else tuple(torch.zeros(tokens, 1, hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    pos, angles = int32([0] * tokens), angles_of(1)
    if how == "cleared":
        acc = x.float()
        got = ops.qkv_append(acc, pos, angles, cache, hq, hkv, scale=3.0, clear=True)
        assert not acc.any()
    else:
        got = ops.qkv_append(x, pos, angles, cache, hq, hkv, scale=3.0, out=x)
        assert got.data_ptr() == x.data_ptr()
    assert torch.equal(got, want)
    k, v = (t.unflatten(1, (hkv, 128)) for t in want[:, hq * 128:].chunk(2, dim=1))
    for i, t in ((0, k), (2 if bits == 4 else 1, v)):
        if bits == 16:
            assert torch.equal(cache[i][:, 0], t)
        else:
            n, s = quantised(t)
            assert torch.equal(codes_of(cache[i])[:, :, 0], n) and torch.equal(cache[i + 1][:, :, 0], s)
    ops.device_status()
