"""Where the result of packed prompt attention lies: rows and heads of `out` on 16-byte boundaries that are not 32-byte ones, with room around them."""
import pytest
import torch

from test_gpu_attn_prompt import check, int32, rand, reference, spans_of, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (6, 2)])
@pytest.mark.parametrize("place", ["heads", "rows", "base"])
@pytest.mark.parametrize("lengths", [[1], [33, 1, 200, 0, 7], [129, 300]], ids=lambda v: "-".join(map(str, v)))
def test_results_on_sixteen_bytes(dtype, d, heads, kv_heads, place, lengths):
    """Ends of items inside a warp's rows, so that some of its lanes have a row to write and some have none.  What lies between the results stays."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(sum(lengths) + heads + d)
    T = sum(lengths) + 2                                       # two rows of no sequence behind the last
    q, k, v = rand(g, (T, heads, d), dtype), rand(g, (T, kv_heads, d), dtype), rand(g, (T, kv_heads, d), dtype)
    if place == "heads":
        whole = torch.full((T, heads, d + 8), 7.0, dtype=dtype, device="cuda")
        out, rest = whole[:, :, :d], whole[:, :, d:]
    elif place == "rows":
        whole = torch.full((T, heads * d + 8), 7.0, dtype=dtype, device="cuda")
        out, rest = whole[:, :heads * d].unflatten(1, (heads, d)), whole[:, heads * d:]
    else:
        whole = torch.full((T * heads * d + 16,), 7.0, dtype=dtype, device="cuda")
        out, rest = whole[8:-8].view(T, heads, d), torch.cat((whole[:8], whole[-8:]))
        assert out.data_ptr() % 32 == 16
    assert ops.attn_prompt(q, k, v, starts_of(lengths), out=out).data_ptr() == out.data_ptr()
    n = T - 2
    check(out[:n], *reference(q[:n], k[:n], v[:n], spans_of(lengths), d ** -0.5))
    rest = torch.cat((whole[:8], whole[-8:])) if place == "base" else rest
    assert (rest == 7).all() and (out[n:] == 7).all()
    assert torch.equal(out[:n], ops.attn_prompt(q, k, v, starts_of(lengths))[:n])      # the bits of a result that lies on 32 bytes
    ops.device_status()


@pytest.mark.parametrize("d", [64, 128])
def test_queries_without_a_key_on_sixteen_bytes(d):
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v = (rand(g, (300, 2, d), torch.float16) for _ in range(3))
    out = torch.full((300, 2, d + 8), 7.0, dtype=torch.float16, device="cuda")[:, :, :d]
    ops.attn_prompt(q, k, v, starts_of([150, 10, 140]), int32([0, 5, 160]), int32([20, 0, 140]), out=out)
    check(out, *reference(q, k, v, [(0, 150, 0, 20), (150, 10, 5, 0), (160, 140, 160, 140)], d ** -0.5))
    assert not out[:130].any() and not out[150:160].any()
