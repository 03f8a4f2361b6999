"""Packed prompt attention where nearly all of a row's weight is on one key and many others share the rest."""
import math

import pytest
import torch

from test_gpu_attn_prompt import int32, rand, reference

pytestmark = pytest.mark.gpu


def small(dtype, keys):
    """What weights below a type's normal numbers may be off by, together, relative to the largest value: fp16 weights are at least 2^7 for the largest score, and half a
    step of fp16's smallest numbers is 2^-25; bf16 has fp32's exponents."""
    return keys * 2.0**-32 if dtype == torch.float16 else 0.0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("below", [14.0, 20.0, 25.5, 28.0])
@pytest.mark.parametrize("at", [0, 30000, 59999])
def test_one_key_and_many_small_ones(dtype, d, below, at):
    """One query over 60000 keys: a score of 16, and all others `below` powers of two less.  The values tell the small ones' share: 0 behind the large one."""
    from rptc_b200 import ops
    n = 60000
    q, k, v = (torch.zeros(s, dtype=dtype, device="cuda") for s in ((1, 1, d), (n, 1, d), (n, 1, d)))
    q[..., 0], k[..., 0], v[:] = 1, 16 - below * math.log(2), 1
    k[at, :, 0], v[at] = 16, 0
    got = ops.attn_prompt(q, k, v, int32([0, 1]), int32([0]), int32([n]), scale=1.0)
    want, tol = reference(q, k, v, [(0, 1, 0, n)], 1.0)
    off = (got.double() - want).abs().max().item()
    print("off %.2e, room %.2e of %.2e" % (off, tol.max().item() + small(dtype, n), want.max().item()))
    assert off <= tol.max().item() + small(dtype, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1)])
def test_a_first_key_that_takes_nearly_all(dtype, heads, kv_heads):
    """Rows of a whole prompt whose first key stands out by 16 to 30 powers of two, values of both signs and a mean."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(heads)
    n, d = 3000, 128
    q, k = rand(g, (n, heads, d), dtype), rand(g, (n, kv_heads, d), dtype)
    v = (1 + torch.randn(n, kv_heads, d, generator=g, device="cuda")).to(dtype)
    q[..., 0], k[..., 0] = torch.linspace(1.1, 1.9, n, device="cuda")[:, None].to(dtype), 0
    k[0, :, :], k[0, :, 0], v[0] = 0, 128.0, 0                  # a score of 128 * 1.1 .. 1.9 / 11.3
    got = ops.attn_prompt(q, k, v, int32([0, n]))
    want, tol = reference(q, k, v, [(0, n, 0, n)], d ** -0.5)
    off = ((got.double() - want).abs() / (tol + small(dtype, n) * v.abs().max().item())).max().item()
    print("off %.2f of the room" % off)
    assert off <= 1
