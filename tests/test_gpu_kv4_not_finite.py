"""Values that are not finite on their way through a 4-bit cache: their groups of 32 stand for NaN, and nothing else does."""
import math

import pytest
import torch

from test_gpu_kv4 import angles_of, codes_of, decoded, int32, quantised

pytestmark = pytest.mark.gpu

BAD = [math.nan, math.inf, -math.inf]


def cached(x, hkv, transform):
    from rptc_b200 import ops
    tokens = len(x)
    cache = ops.kv4_cache(tokens, 1, hkv)
    out = ops.qkv_append(x, int32([0] * tokens), angles_of(1), cache, hkv, hkv, transform=transform)
    ops.device_status()
    return out, cache


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("bad", [[b] for b in BAD] + [[math.nan, math.inf], [math.inf, -math.inf], [math.inf] * 32, [-math.inf] * 32, [math.nan] * 32], ids=str)
@pytest.mark.parametrize("at", [0, 5, 31, 64, 96, 127])
def test_a_group_with_such_a_value(dtype, bad, at):
    """One group of one head of v, wherever in it they are; of k that of the rotation's partners too, 64 values on, which is infinite times a sine of 0."""
    g = torch.Generator(device="cuda").manual_seed(at)
    hkv = 3
    x = torch.randn(4, 3 * hkv * 128, generator=g, device="cuda").half().to(dtype)
    for head in (hkv + 1, 2 * hkv + 2):                        # of k and of v
        first = head * 128 + (at if len(bad) < 32 else at // 32 * 32)
        x[2, first:first + len(bad)] = torch.tensor(bad, device="cuda").to(dtype)[:(head + 1) * 128 - first]      # behind the head's last value: the next one's
    out, cache = cached(x, hkv, False)
    assert torch.equal(out[[0, 1, 3]], x.half()[[0, 1, 3]])
    for i, part in ((0, out[:, hkv * 128:2 * hkv * 128]), (2, out[:, 2 * hkv * 128:])):
        part = part.unflatten(1, (hkv, 128))
        lost = ~part.unflatten(2, (4, 32)).isfinite().all(-1)
        given = ~x[:, (hkv if i == 0 else 2 * hkv) * 128:].half()[:, :hkv * 128].unflatten(1, (hkv, 4, 32)).isfinite().all(-1)
        assert given.any() and torch.equal(lost, given | given.roll(2, -1) if i == 0 else given)
        held = decoded(cache[i], cache[i + 1])[:, :, 0].unflatten(2, (4, 32))
        assert held[lost].isnan().all() and held[~lost].isfinite().all()
        n, s = quantised(torch.where(lost[..., None].expand(-1, -1, -1, 32).flatten(2), 0, part))
        assert torch.equal(codes_of(cache[i])[:, :, 0].unflatten(2, (4, 32))[~lost], n.unflatten(2, (4, 32))[~lost])
        assert torch.equal(cache[i + 1][:, :, 0][~lost], s[~lost])


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("hkv,tokens", [(32, 70), (5, 3000)])
def test_tokens_with_such_values_among_many(bad, hkv, tokens):
    """As many as take the transform on the tensor core, which spreads a value over its head of 128."""
    g = torch.Generator(device="cuda").manual_seed(hkv)
    x = torch.randn(tokens, 3 * hkv * 128, generator=g, device="cuda").half()
    clean = cached(x, hkv, True)[1]
    hit = torch.rand(tokens, 3 * hkv, generator=g, device="cuda") < 0.1
    x.unflatten(1, (3 * hkv, 128))[..., 77][hit] = bad
    cache = cached(x, hkv, True)[1]
    for i, heads in ((0, hit[:, hkv:2 * hkv]), (2, hit[:, 2 * hkv:])):
        held = decoded(cache[i], cache[i + 1])[:, :, 0]
        assert held[heads].isnan().all() and held[~heads].isfinite().all()
        assert torch.equal(cache[i][~heads], clean[i][~heads]) and torch.equal(cache[i + 1][~heads], clean[i + 1][~heads])


@pytest.mark.parametrize("context,max_pos", [(40, 64), (3000, 5000)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_what_reads_the_cache_shows_it(context, max_pos, which):
    """kv4_values and single-token attention, as over an fp16 cache with NaN in the group's place: of a key the whole of a head's result, of a value
    its group of dims; behind the last position nothing."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(context)
    rows, hkv, heads, group = 3, 2, 8, 2
    cache = ops.kv4_cache(rows, max_pos, hkv)
    n = rows * max_pos
    x = torch.randn(n, 3 * hkv * 128, generator=g, device="cuda").half()
    slots, pos = torch.arange(n, device="cuda").int() // max_pos, torch.arange(n, device="cuda").int() % max_pos
    at = (hkv + 1 if which == "k" else 2 * hkv + 1) * 128 + 32 * group + 9
    x[max_pos + context // 2, at] = math.inf                   # row 1, kv head 1
    x[2 * max_pos + context, at] = math.nan                    # row 2, behind its last position
    angles = torch.zeros(max_pos, 64, 2, device="cuda")
    angles[..., 0] = 1                                          # no rotation: a value stays in its group, but for the partner that is infinite times 0
    lost = [group, group - 2] if which == "k" else [group]
    ops.qkv_append(x, pos, angles, cache, hkv, hkv, slots=slots)
    values = ops.kv4_values(cache, int32([max_pos] * rows))
    for t, name in zip(values, "kv"):
        want = torch.zeros_like(t, dtype=torch.bool)
        if name == which:
            for r, p in ((1, context // 2), (2, context)):
                for j in lost:
                    want[r, p, 1, 32 * j:32 * j + 32] = True
        assert torch.equal(t.isnan(), want) and t[~want].isfinite().all()
    q = torch.randn(rows, heads * 128, generator=g, device="cuda").half()
    got = ops.attn_decode_kv4(q, int32([context - 1] * rows), cache, heads).unflatten(1, (hkv, heads // hkv, 4, 32))
    want = torch.zeros_like(got, dtype=torch.bool)
    want[1, 1, :, slice(None) if which == "k" else group] = True
    assert torch.equal(got.isnan(), want) and got[~want].isfinite().all()
    ops.device_status()
