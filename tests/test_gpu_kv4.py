"""The KV cache in 4 bits: append (ops.qkv_append), the values it stands for (ops.kv4_values) and single-token attention over it
(ops.attn_decode_kv4), against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def angles_of(n):
    inv = 10000.0 ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack((a.cos(), a.sin()), -1).float().contiguous()


def hadamard(x):
    """orthonormal, along the last axis of 128, in 64 bits"""
    h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for _ in range(7):
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return x @ h / math.sqrt(128)


def place():
    """byte and shift of a position's 128 values in its 64 bytes"""
    e, g = torch.arange(128, device="cuda") % 32, torch.arange(128, device="cuda") // 32
    return 2 * (4 * (e // 4) + g) + (e % 4) // 2, 4 * (e % 2), g


def decoded(codes, scales):
    """the values that codes [..., 64] and scales [..., 4, 2] stand for, 64 bits"""
    byte, shift, g = place()
    return scales[..., g, 1].double() + ((codes[..., byte].long() >> shift) & 15).double() * scales[..., g, 0].double()


def quantised(x):
    """codes [..., 128] and scales of fp16 values, 64 bits up to the two roundings that the format has"""
    g = x.double().unflatten(-1, (4, 32))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low) / 15).half()
    step = scale.double()[..., None]
    n = torch.where(step > 0, ((g - low[..., None]) / step).round().clamp(max=15), 0.0)      # torch.round: half to even
    return n.flatten(-2).long(), torch.stack((scale, low.half()), -1)


def codes_of(codes):
    byte, shift, _ = place()
    return (codes[..., byte].long() >> shift) & 15


def random_cache(g, rows, max_pos, kv_heads, spread=1.0, offset=0.0):
    from rptc_b200 import ops
    cache = ops.kv4_cache(rows, max_pos, kv_heads)
    for i in (0, 2):
        cache[i].copy_(torch.randint(0, 256, cache[i].shape, generator=g, device="cuda", dtype=torch.uint8))
        scale = spread * (0.1 + 0.3 * torch.rand(cache[i + 1].shape[:-1], generator=g, device="cuda"))
        cache[i + 1].copy_(torch.stack((scale, offset - 7.5 * scale + spread * torch.randn(scale.shape, generator=g, device="cuda")), -1).half())
    return cache


# ---- append --------------------------------------------------------------------------------------------------------------
def finished(x, signs, scale, transform, angles, pos, hq, hkv):
    """q, k, v as they should leave, in 64 bits with the fp16 rounding in the middle, and how far a kernel may be off: its own rounding, and in front of
    the rotation a neighbour of the rounded value (a step, 2^-10) where 32 bits decide otherwise than 64.  The transform's 32-bit error is not relative to its
    result: each of its seven stages rounds a sum that is at most sum |x| by 2^-24 of that, and later stages add up what all 128 / 2^stage partial sums are off, which again is
    2^-24 of sum |x| at most: seven stages, and the scale's rounding, are 8 * 2^-24 * sum |x| * scale / sqrt(128) for each of the rotation's two values."""
    y = x.double().unflatten(1, (hq + 2 * hkv, 128))
    lost = 8 * 2.0**-24 * y.abs().sum(-1, keepdim=True) * scale / math.sqrt(128) if transform else 0.0
    if transform:
        y = hadamard(y)
        if signs is not None:
            y = y * signs.double().unflatten(0, (-1, 128))
    y = (y * scale).half().double()
    cs, sn = (angles[pos.long()][:, None, :, i].double() for i in (0, 1))
    a, b = y[..., :64], y[..., 64:]
    turned = torch.cat((a * cs - b * sn, a * sn + b * cs), -1)
    room = torch.cat((a.abs() + b.abs(),) * 2, -1)
    turned[:, hq + hkv:], room[:, hq + hkv:] = y[:, hq + hkv:], y[:, hq + hkv:].abs()
    return turned, 2.0**-11 * turned.abs() + 2.0**-10 * room + 2.0**-24 + 2 * lost


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("transform", [True, False])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 2), (9, 3), (32, 32)])
def test_append(bits, dtype, transform, hq, hkv):
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(hq)
    rows, max_pos, tokens, width = 5, 70, 37, (hq + 2 * hkv) * 128
    x = (3 * torch.randn(tokens, width + 8, generator=g, device="cuda")).to(dtype)[:, :width]
    signs = (torch.randint(0, 2, (width,), generator=g, device="cuda") * 2 - 1).half() if transform else None
    spot = torch.randperm(rows * max_pos, generator=g, device="cuda")[:tokens]
    slots, pos = (spot // max_pos).int(), (spot % max_pos).int()
    angles = angles_of(max_pos + 3)
    cache = ops.kv4_cache(rows, max_pos, hkv) if bits == 4 else tuple(torch.zeros(rows, max_pos, hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    before = x.clone()
    out = ops.qkv_append(x, pos, angles, cache, hq, hkv, slots=slots, signs_out=signs, scale=0.25, transform=transform)
    assert torch.equal(x, before)
    want, tol = finished(x, signs, 0.25, transform, angles, pos, hq, hkv)
    got = out.unflatten(1, (-1, 128))
    off = ((got.double() - want).abs() / tol).max().item()
    assert off <= 1, off
    k, v = got[:, hq:hq + hkv], got[:, hq + hkv:]
    seen = torch.zeros(rows * max_pos, dtype=torch.bool, device="cuda")
    seen[spot] = True
    seen = seen.view(rows, max_pos)
    if bits == 16:
        assert torch.equal(cache[0][slots.long(), pos.long()], k) and torch.equal(cache[1][slots.long(), pos.long()], v)
        assert not cache[0][~seen].any() and not cache[1][~seen].any()
    else:
        for i, t in ((0, k), (2, v)):
            n, s = quantised(t)
            assert torch.equal(codes_of(cache[i])[slots.long(), :, pos.long()], n)
            assert torch.equal(cache[i + 1][slots.long(), :, pos.long()], s)
            assert not cache[i].transpose(1, 2)[~seen].any() and not cache[i + 1].transpose(1, 2)[~seen].any()
    ops.device_status()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("hq,hkv,tokens", [(32, 32, 70), (12, 4, 401), (64, 8, 300), (16, 2, 1000), (5, 5, 3000), (40, 20, 77)])
def test_append_of_many_tokens(bits, hq, hkv, tokens):
    """Enough tokens of fp16 for the transform on the tensor core, whose sums of sixteen take the place of four of the seven stages: each is within 4 * 2^-24 of its
    sum |x|.  Eights that are full, and not; values of all sizes; tokens of no sequence; in place, and q alone."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rows, max_pos, width = 7, tokens // 5, (hq + 2 * hkv) * 128
    size = torch.tensor([3.0, 0.01, 2e-6, 100.0, 0.0, 1e-4, 0.5], device="cuda")[torch.arange(tokens, device="cuda") % 7]
    x = torch.zeros(tokens, width + 8, dtype=torch.float16, device="cuda")[:, :width].copy_(size[:, None] * torch.randn(tokens, width, generator=g, device="cuda"))
    signs = (torch.randint(0, 2, (width,), generator=g, device="cuda") * 2 - 1).half()
    spot = torch.randperm(rows * max_pos, generator=g, device="cuda")[:tokens]
    slots, pos = (spot // max_pos).int(), (spot % max_pos).int()
    idle = torch.arange(tokens, device="cuda") % 11 == 3
    pos[idle] = -1
    angles = angles_of(max_pos)
    new = lambda: ops.kv4_cache(rows, max_pos, hkv) if bits == 4 else tuple(torch.zeros(rows, max_pos, hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    cache, again = new(), new()
    out = torch.full((tokens, width), 7.0, dtype=torch.float16, device="cuda")
    assert ops.qkv_append(x, pos, angles, cache, hq, hkv, slots=slots, signs_out=signs, scale=0.25, transform=True, out=out) is out
    assert (out[idle] == 7).all()
    want, tol = finished(x, signs, 0.25, True, angles, pos.clamp(min=0), hq, hkv)
    got = out.unflatten(1, (-1, 128))
    assert ((got.double() - want).abs() <= tol)[~idle].all(), ((got.double() - want).abs() / tol)[~idle].max()
    k, v, at = got[~idle, hq:hq + hkv], got[~idle, hq + hkv:], (slots[~idle].long(), pos[~idle].long())
    seen = torch.zeros(rows, max_pos, dtype=torch.bool, device="cuda")
    seen[at] = True
    if bits == 16:
        assert torch.equal(cache[0][at], k) and torch.equal(cache[1][at], v) and not cache[0][~seen].any() and not cache[1][~seen].any()
    else:
        for i, t in ((0, k), (2, v)):
            n, s = quantised(t)
            assert torch.equal(codes_of(cache[i])[at[0], :, at[1]], n) and torch.equal(cache[i + 1][at[0], :, at[1]], s)
            assert not cache[i].transpose(1, 2)[~seen].any() and not cache[i + 1].transpose(1, 2)[~seen].any()
    q = torch.full((tokens, hq * 128), 7.0, dtype=torch.float16, device="cuda")
    ops.qkv_append(x, pos, angles, again, hq, hkv, slots=slots, signs_out=signs, scale=0.25, transform=True, out=q)
    assert torch.equal(q, out[:, :hq * 128]) and all(torch.equal(a, b) for a, b in zip(cache, again))
    held = x.clone()
    ops.qkv_append(x, pos, angles, again, hq, hkv, slots=slots, signs_out=signs, scale=0.25, transform=True, out=x)
    assert torch.equal(x[~idle], out[~idle]) and torch.equal(x[idle], held[idle]) and all(torch.equal(a, b) for a, b in zip(cache, again))
    ops.device_status()


def test_append_q_alone_in_place_and_cleared():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    hq, hkv, width = 4, 2, 8 * 128
    x = torch.randn(3, width, generator=g, device="cuda")
    pos, angles = int32([4, 0, 9]), angles_of(10)
    a, b, c = (ops.kv4_cache(3, 10, hkv) for _ in range(3))
    full = ops.qkv_append(x, pos, angles, a, hq, hkv, transform=True)
    q = torch.full((3, hq * 128 + 8), 5.0, dtype=torch.float16, device="cuda")
    acc = x.clone()
    ops.qkv_append(acc, pos, angles, b, hq, hkv, transform=True, out=q[:, :hq * 128], clear=True)
    assert torch.equal(q[:, :hq * 128], full[:, :hq * 128]) and (q[:, hq * 128:] == 5).all() and not acc.any()
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    h = x.half()
    want = ops.qkv_append(h, pos, angles, a, hq, hkv, transform=True)
    got = ops.qkv_append(h, pos, angles, c, hq, hkv, transform=True, out=h)
    assert got.data_ptr() == h.data_ptr() and torch.equal(got, want) and all(torch.equal(s, t) for s, t in zip(a, c))


def test_append_values_of_all_sizes():
    """Groups that are constant, tiny, huge, and with ties half-way between two codes."""
    from rptc_b200 import ops
    rows = [torch.zeros(128), torch.full((128,), 3.7), torch.linspace(-1, 1, 128) * 6e-8, torch.linspace(-65504, 65504, 128), torch.arange(128) % 32 * 0.5,
            torch.cat((torch.tensor([0.0, 15.0]), torch.arange(126) % 15 + 0.5)), torch.arange(128) * 2.0**-24, -torch.arange(128.0) ** 3]
    x = torch.stack([torch.cat((torch.zeros(128), t, t)) for t in rows]).half().cuda()
    cache = ops.kv4_cache(len(rows), 1, 1)
    angles = angles_of(1)                                     # position 0: no rotation
    out = ops.qkv_append(x, int32([0] * len(rows)), angles, cache, 1, 1)
    # the last row's cubes pass fp16's range: it holds infinities, which stand for no code; its neighbours do not notice
    assert x[-1].isinf().any() and x[:-1].isfinite().all()
    out, x, cache = out[:-1], x[:-1], [t[:-1] for t in cache]
    assert torch.equal(out, x)
    for i in (0, 2):
        n, s = quantised(x[:, 128:256])
        assert torch.equal(codes_of(cache[i])[:, 0, 0], n) and torch.equal(cache[i + 1][:, 0, 0], s)
        assert ((decoded(cache[i], cache[i + 1])[:, 0, 0] - x[:, 128:256].double()).abs().unflatten(1, (4, 32)) <= s[..., :1].double() * (0.5 + 15 * 2.0**-11) + 15 * 2.0**-25).all()


def test_append_skips_tokens_of_no_sequence_and_reports_positions_outside():
    from rptc_b200 import RPTCError, ops
    x = torch.randn(4, 3 * 128, device="cuda")
    angles = angles_of(8)
    ops.device_status()
    cache = ops.kv4_cache(4, 8, 1)
    out = torch.full((4, 3 * 128), 9.0, dtype=torch.float16, device="cuda")
    acc = x.clone()
    ops.qkv_append(acc, int32([0, -1, 7, -1]), angles, cache, 1, 1, out=out, clear=True)
    ops.device_status()
    assert (out[1] == 9).all() and (out[3] == 9).all() and not acc.any()
    assert not cache[1][1].any() and not cache[1][3].any() and cache[1][0, 0, 0].any() and cache[1][2, 0, 7].any()
    for pos, slots in (([8, 0, 0, 0], None), ([-2, 0, 0, 0], None), ([0, 0, 0, 0], [0, 1, 2, 4]), ([0, 0, 0, 0], [-1, 1, 2, 3])):
        ops.qkv_append(x, int32(pos), angles, cache, 1, 1, slots=None if slots is None else int32(slots))
        with pytest.raises(RPTCError):
            ops.device_status()


# ---- values --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,max_pos,hkv", [(1, 1, 1), (3, 77, 2), (2, 1000, 8)])
def test_values(rows, max_pos, hkv):
    from rptc_b200 import RPTCError, ops
    g = torch.Generator(device="cuda").manual_seed(max_pos)
    cache = random_cache(g, rows, max_pos, hkv)
    count = [max_pos, 0, max_pos // 2][:rows]
    out = tuple(torch.full((rows, max_pos, hkv, 128), 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv4_values(cache, int32(count), out)
    for i, t in ((0, out[0]), (2, out[1])):
        want = decoded(cache[i], cache[i + 1]).half().transpose(1, 2)
        for r, n in enumerate(count):
            # code * scale and the sum are exact in 32 bits or rounded far below fp16: the same fp16, or its neighbour at a tie
            assert ((t[r, :n].double() - want[r, :n].double()).abs() <= 2.0**-10 * want[r, :n].abs().double() * 2.0**-10 + (2.0**-11 + 2.0**-20) * want[r, :n].abs().double() + 2.0**-25).all()
            assert (t[r, n:] == 3).all()
    ops.device_status()
    for bad in (-1, max_pos + 1):
        ops.kv4_values(cache, int32([bad] + [0] * (rows - 1)), out)
        with pytest.raises(RPTCError):
            ops.device_status()


# ---- attention -----------------------------------------------------------------------------------------------------------
def reference(q, pos, cache, heads, scale):
    """The result in 64 bits, and how far a kernel may be off: the result's rounding; 2^-11 for a weight times a group's scale in fp16, on codes counted
    from the middle (at most 8 scales); and in units of 32 bits, relative to the sums of |weight| times the largest that a code and a minimum can be apart: the
    scores' sums of 128 products (of codes to 15 and minimums, hence the larger sizes), sums over the positions, exp2."""
    rows, hkv, max_pos = cache[0].shape[:3]
    out, tol = (torch.zeros(rows, heads, 128, dtype=torch.float64, device="cuda") for _ in range(2))
    for r, n in enumerate((pos + 1).tolist()):
        for h in range(heads if n else 0):
            c = h // (heads // hkv)
            k, v = (decoded(cache[i][r, c, :n], cache[i + 1][r, c, :n]) for i in (0, 2))
            ks, vs = (cache[i][r, c, :n].double().repeat_interleave(32, dim=1) for i in (1, 3))
            x = q[r, h * 128:(h + 1) * 128].double()
            p = (scale * (k @ x)).softmax(0)
            score = scale * ((ks[..., 1].abs() + 15 * ks[..., 0]) @ x.abs()).max()
            eighth = p @ (8 * vs[..., 0])
            out[r, h] = p @ v
            tol[r, h] = 2.0**-11 * (out[r, h].abs() + eighth) + (score * 128 * 2.0**-23 + 2 * n * 2.0**-24 + 2.0**-18) * (p @ (vs[..., 1].abs() + 15 * vs[..., 0])) + 2.0**-25
    return out, tol


def check(got, q, pos, cache, heads, scale=128 ** -0.5):
    want, tol = reference(q, pos, cache, heads, scale)
    got = got.unflatten(1, (heads, 128)).double()
    assert got.isfinite().all()
    off = ((got - want).abs() / tol.clamp(min=1e-30)).max().item()
    print("max err/tol %.3f" % off)
    assert off <= 1


@pytest.mark.parametrize("heads,hkv", [(4, 4), (8, 1), (6, 2), (16, 2), (5, 1), (24, 2), (32, 1)])
@pytest.mark.parametrize("max_pos,pos", [(1, [0]), (70, [0, 1, 15, 16, 63, 64, 69]), (600, [599, 300, 127, 128]), (2100, [2047, 2099])])
def test_attention(heads, hkv, max_pos, pos):
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(heads + max_pos)
    cache = random_cache(g, len(pos), max_pos, hkv)
    for t in cache[1], cache[3]:                               # what lies behind a row's position does not matter
        for r, n in enumerate(pos):
            t[r, :, n + 1:] = math.nan
    q = torch.randn(len(pos), heads * 128, generator=g, device="cuda").half()
    got = ops.attn_decode_kv4(q, int32(pos), cache, heads)
    check(got, q, int32(pos), cache, heads)
    assert torch.equal(got, ops.attn_decode_kv4(q, int32(pos), cache, heads))
    ops.device_status()


@pytest.mark.parametrize("heads,hkv,rows,context", [(8, 1, 1, 40000), (64, 8, 3, 5001), (4, 4, 1, 9000)])
def test_attention_over_long_contexts(heads, hkv, rows, context):
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(context)
    cache = random_cache(g, rows, context + 5, hkv)
    q = torch.randn(rows, heads * 128, generator=g, device="cuda").half()
    pos = int32([context - 1 - 700 * r for r in range(rows)])
    check(ops.attn_decode_kv4(q, pos, cache, heads), q, pos, cache, heads)


@pytest.mark.parametrize("heads,hkv,rows,max_pos,most", [(8, 8, 40, 2100, 2100), (64, 4, 40, 2100, 700), (2, 1, 300, 2049, 90), (3, 3, 100, 2304, 2304), (8, 8, 36, 2500, 40), (8, 2, 70, 4000, 1)])
def test_attention_of_many_rows(heads, hkv, rows, max_pos, most):
    """More items than ranges, and fewer: lengths of all sizes, rows of no sequence among them, a range's end at any place of an item."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    cache = random_cache(g, rows, max_pos, hkv)
    q = torch.randn(rows, heads * 128, generator=g, device="cuda").half()
    pos = torch.randint(-1, most, (rows,), generator=g, device="cuda", dtype=torch.int32)
    pos[0], pos[rows - 1] = most - 1, -1
    for r, n in enumerate(pos.tolist()):
        for t in cache[1], cache[3]:
            t[r, :, n + 1:] = math.nan
    got = ops.attn_decode_kv4(q, pos, cache, heads)
    check(got, q, pos, cache, heads)
    assert (got[pos < 0] == 0).all()
    for last in (0, rows // 2, rows - 1):                      # one row alone
        alone = torch.full_like(pos, -1)
        alone[last] = most - 1
        for t in cache[1], cache[3]:
            t[last].nan_to_num_(nan=0.5)
        check(ops.attn_decode_kv4(q, alone, cache, heads), q, alone, cache, heads)
    assert (ops.attn_decode_kv4(q, torch.full_like(pos, -1), cache, heads) == 0).all()
    ops.device_status()


def test_attention_of_a_few_rows_among_idle_ones():
    """A range's next item may be hundreds of rows on."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = random_cache(g, 400, 2200, 2)
    q = torch.randn(400, 4 * 128, generator=g, device="cuda").half()
    for rows in ([0, 1, 399], [31, 32, 95, 96, 300], [399], [7] + list(range(200, 330))):
        pos = torch.full((400,), -1, dtype=torch.int32, device="cuda")
        pos[rows] = torch.randint(0, 2200, (len(rows),), generator=g, device="cuda", dtype=torch.int32)
        got = ops.attn_decode_kv4(q, pos, cache, 4)
        check(got, q, pos, cache, 4)
        assert (got[pos < 0] == 0).all()
    ops.device_status()


@pytest.mark.parametrize("spread,offset,q_spread,scale", [(1e-4, 0, 1, None), (300, 0, 0.1, 1e-3), (1, 50, 1, None), (1, 0, 40, None), (1, 0, 1e-4, 1.0), (0.0, 2.0, 1, None),
                                                          (1, 0, 1000, 1e-2)])
def test_values_of_all_sizes(spread, offset, q_spread, scale):
    """Small and large scales, all values in a group equal (scale 0), weights nearly all on one position."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(17)
    cache = random_cache(g, 2, 333, 2, spread, offset)
    q = (q_spread * torch.randn(2, 8 * 128, generator=g, device="cuda")).half()
    pos = int32([332, 40])
    scale = 128 ** -0.5 if scale is None else scale
    check(ops.attn_decode_kv4(q, pos, cache, 8, scale=scale), q, pos, cache, 8, scale)


def test_scales_that_differ_from_position_to_position():
    """The largest weight on values with the smallest scale, and the other way round."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(18)
    cache = random_cache(g, 1, 500, 1)
    size = (2.0 ** torch.arange(-14, 6, device="cuda").float()).repeat(25)
    cache[3][0, 0] = (cache[3][0, 0].float() * size[:, None, None]).half()
    cache[1][0, 0] = (cache[1][0, 0].float() * (3 * size.flip(0).clamp(max=1))[:, None, None]).half()
    q = torch.randn(1, 4 * 128, generator=g, device="cuda").half()
    check(ops.attn_decode_kv4(q, int32([499]), cache, 4), q, int32([499]), cache, 4)


def test_rows_of_no_sequence_and_positions_outside():
    from rptc_b200 import RPTCError, ops
    g = torch.Generator(device="cuda").manual_seed(19)
    cache = random_cache(g, 3, 50, 2)
    q = torch.randn(3, 4 * 128, generator=g, device="cuda").half()
    ops.device_status()
    pos = int32([20, -1, 49])
    out = torch.full((3, 4 * 128), 9.0, dtype=torch.float16, device="cuda")
    ops.attn_decode_kv4(q, pos, cache, 4, out=out)
    ops.device_status()
    assert not out[1].any()
    check(out, q, pos, cache, 4)
    for bad in (-2, 50):
        got = ops.attn_decode_kv4(q, int32([20, bad, 49]), cache, 4)
        with pytest.raises(RPTCError):
            ops.device_status()
        assert not got[1].any() and torch.equal(got[0], out[0]) and torch.equal(got[2], out[2])


def test_output_transform_and_strides():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(20)
    cache = random_cache(g, 2, 200, 2)
    buf = torch.randn(2, 12 * 128, generator=g, device="cuda").half()      # a fused buffer whose first heads are q
    pos = int32([199, 77])
    signs = (torch.randint(0, 2, (8 * 128,), generator=g, device="cuda") * 2 - 1).half()
    plain = ops.attn_decode_kv4(buf[:, :8 * 128].contiguous(), pos, cache, 8)
    out = torch.full((2, 9 * 128), 9.0, dtype=torch.float16, device="cuda")
    ops.attn_decode_kv4(buf, pos, cache, 8, out=out)
    assert torch.equal(out[:, :8 * 128], plain) and (out[:, 8 * 128:] == 9).all()
    got = ops.attn_decode_kv4(buf, pos, cache, 8, signs_in=signs)
    want = hadamard((plain.double() * signs.double()).unflatten(1, (8, 128)))
    # the plain output is rounded once more in front of the transform than it need be: 2^-11 of each of 128 values over sqrt(128), twice; and the result
    room = 2 * 2.0**-11 * plain.double().abs().unflatten(1, (8, 128)).sum(-1, keepdim=True) / math.sqrt(128) + 2.0**-11 * want.abs() + 2.0**-20
    assert ((got.double().unflatten(1, (8, 128)) - want).abs() <= room).all()


def test_captured_call_follows_the_positions_and_two_graphs_run_at_once():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(21)
    cache = random_cache(g, 2, 3000, 2)
    q = torch.randn(2, 4 * 128, generator=g, device="cuda").half()
    graphs = []
    for _ in range(2):
        pos, out, stream = int32([0, 0]), torch.zeros(2, 4 * 128, dtype=torch.float16, device="cuda"), torch.cuda.Stream()
        ops.attn_decode_kv4(q, pos, cache, 4, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.attn_decode_kv4(q, pos, cache, 4, out=out)
        graphs.append((graph, pos, out, stream))
    for spots in (([0, 5], [2999, 1]), ([100, 2999], [64, 63]), ([2000, 2000], [500, -1])):
        for (graph, pos, out, stream), p in zip(graphs, spots):
            pos.copy_(int32(p))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, pos, out, stream in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, pos, out, stream in graphs:
            check(out, q, pos, cache, 4)


def test_append_then_attention_under_dependent_launch():
    """A decode step's two calls behind one another, as the engine queues them: the new position takes part."""
    from rptc_b200 import lib, ops
    g = torch.Generator(device="cuda").manual_seed(22)
    hq, hkv, rows = 8, 2, 4
    angles = angles_of(64)
    plain, chained = ops.kv4_cache(rows, 64, hkv), ops.kv4_cache(rows, 64, hkv)
    steps = [torch.randn(rows, (hq + 2 * hkv) * 128, generator=g, device="cuda") for _ in range(40)]
    want = []
    for t, x in enumerate(steps):
        pos = int32([t] * rows)
        out = ops.qkv_append(x, pos, angles, plain, hq, hkv, transform=True)
        torch.cuda.synchronize()
        want.append(ops.attn_decode_kv4(out, pos, plain, hq))
        torch.cuda.synchronize()
        check(want[-1], out, pos, plain, hq)
    places = [int32([t] * rows) for t in range(40)]
    torch.cuda.synchronize()
    lib().rptc_set_pdl(1)
    try:
        got = [ops.attn_decode_kv4(ops.qkv_append(x, p, angles, chained, hq, hkv, transform=True), p, chained, hq) for x, p in zip(steps, places)]
    finally:
        lib().rptc_set_pdl(0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
