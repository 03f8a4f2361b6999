"""Causal attention of packed prompts (ops.attn_prompt) against the formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(lengths, first=0):
    return int32([first + sum(lengths[:i]) for i in range(len(lengths) + 1)])


def rand(g, shape, dtype, spread=1.0):
    return (spread * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def reference(q, k, v, spans, scale):
    """spans: (q0, n, k0, m) of each sequence.  Returns the result in 64 bits and how far a kernel may be off:
    the result's rounding, that of each weight (half a step of the type, relative to it), and in units of 32 bits, relative to sum p |v|: an error of a
    score is one of its weight, a score is a sum of d products, a result a sum of m, the total of the weights too; 2^-19 for exp2 and
    the scores' scaling."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda")
    tol = out.clone()
    u = torch.finfo(q.dtype).eps / 2
    group = q.shape[1] // k.shape[1]
    for q0, n, k0, m in spans:
        for h in range(q.shape[1]):
            a, b, c = q[q0:q0 + n, h].double(), k[k0:k0 + m, h // group].double(), v[k0:k0 + m, h // group].double()
            seen = torch.arange(m, device="cuda") <= (m - n + torch.arange(n, device="cuda"))[:, None]
            p = torch.where(seen, scale * (a @ b.t()), -math.inf).softmax(-1)
            p = torch.where(seen, p, 0.0)                      # a row that sees nothing: zeros
            score = (scale * (a.abs() @ b.abs().t()) * seen).amax(-1, keepdim=True) if m else torch.zeros(n, 1, device="cuda", dtype=torch.float64)
            weighed = p @ c.abs()
            out[q0:q0 + n, h] = p @ c
            tol[q0:q0 + n, h] = u * out[q0:q0 + n, h].abs() + (u + score * q.shape[2] * 2.0**-23 + 2 * m * 2.0**-24 + 2.0**-19) * weighed + 2.0**-25
    return out, tol


def check(got, want, tol, what=""):
    there = ~want.isnan()
    assert got[there].isfinite().all(), what
    off = ((got.double() - want).abs() / tol)[there]
    if off.numel():
        print(what, "max err/tol %.3f" % off.max().item())
        assert off.max() <= 1, (what, off.max().item())


def spans_of(lengths, past=None):
    past = past or [0] * len(lengths)
    spans, q0, k0 = [], 0, 0
    for n, p in zip(lengths, past):
        spans.append((q0, n, k0, n + p))
        q0, k0 = q0 + n, k0 + n + p
    return spans


HEADS = [(4, 4), (8, 1), (6, 2), (16, 2), (5, 1)]
LENGTHS = [[1], [2, 1, 1], [127], [128], [129, 3], [255, 256, 257], [300, 0, 17, 0, 64], [5] * 9, [700], [1000, 31]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "-".join(map(str, v)))
def test_packed_prompts(dtype, d, heads, kv_heads, lengths):
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(sum(lengths) + heads + d)
    T = sum(lengths)
    q, k, v = rand(g, (T, heads, d), dtype), rand(g, (T, kv_heads, d), dtype), rand(g, (T, kv_heads, d), dtype)
    got = ops.attn_prompt(q, k, v, starts_of(lengths))
    check(got, *reference(q, k, v, spans_of(lengths), d ** -0.5))
    assert torch.equal(got, ops.attn_prompt(q, k, v, starts_of(lengths)))      # the same bits again
    ops.device_status()


@pytest.mark.parametrize("d,heads,kv_heads", [(128, 8, 1), (128, 4, 4), (64, 6, 2)])
@pytest.mark.parametrize("lengths,past", [([1], [1]), ([1, 1, 1], [127, 128, 300]), ([40, 7, 0, 200], [100, 0, 50, 513]), ([130], [1025])])
def test_prompts_that_continue(d, heads, kv_heads, lengths, past):
    """Keys in another place and order than the queries, among rows that belong to nobody and hold no numbers."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(d + sum(past))
    T, slot = sum(lengths), max(a + b for a, b in zip(lengths, past)) + 3
    n = len(lengths)
    k, v = (torch.full((n * slot, kv_heads, d), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    q = rand(g, (T, heads, d), torch.float16)
    spans, first, count, q0 = [], [], [], 0
    for s, (a, b) in enumerate(zip(lengths, past)):
        k0 = (n - 1 - s) * slot                                # the last sequence's keys in front
        k[k0:k0 + a + b], v[k0:k0 + a + b] = rand(g, (a + b, kv_heads, d), torch.float16), rand(g, (a + b, kv_heads, d), torch.float16)
        spans.append((q0, a, k0, a + b))
        first.append(k0)
        count.append(a + b)
        q0 += a
    got = ops.attn_prompt(q, k, v, starts_of(lengths), int32(first), int32(count))
    check(got, *reference(q, k, v, spans, d ** -0.5))
    ops.device_status()


def test_queries_without_a_key_give_zeros():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (rand(g, (300, 2, 128), torch.float16) for _ in range(3))
    lengths, count = [150, 10, 140], [20, 0, 140]
    got = ops.attn_prompt(q, k, v, starts_of(lengths), int32([0, 5, 160]), int32(count))
    want, tol = reference(q, k, v, [(0, 150, 0, 20), (150, 10, 5, 0), (160, 140, 160, 140)], 128 ** -0.5)
    check(got, want, tol)
    assert not got[:130].any() and not got[150:160].any()


def test_rows_of_no_sequence_stay_and_do_not_matter():
    """A padded batch: rows in front of, and behind the sequences hold NaN in q, k and v; out keeps what it held."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(4)
    T, lengths = 500, [33, 1, 250]
    q, k, v = (torch.full((T, h, 128), math.nan, dtype=torch.float16, device="cuda") for h in (4, 2, 2))
    for t in (q, k, v):
        t[7:291] = rand(g, (284,) + t.shape[1:], torch.float16)
    out = torch.full_like(q, 7.0)
    back = ops.attn_prompt(q, k, v, starts_of(lengths, 7), out=out)
    assert back.data_ptr() == out.data_ptr()
    check(out[7:291], *reference(q[7:291], k[7:291], v[7:291], spans_of(lengths), 128 ** -0.5))
    assert (out[:7] == 7).all() and (out[291:] == 7).all()


def test_a_neighbour_without_numbers():
    """Infinities and NaN in one sequence stay in it, whatever tile its neighbours share with it."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    lengths = [100, 60, 90]
    q, k, v = (rand(g, (250, 2, 128), torch.float16) for _ in range(3))
    want, tol = reference(q, k, v, spans_of(lengths), 128 ** -0.5)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[100:160], v2[100:160] = bad, bad
        got = ops.attn_prompt(q, k2, v2, starts_of(lengths))
        check(got[:100], want[:100], tol[:100])
        check(got[160:], want[160:], tol[160:])


@pytest.mark.parametrize("layout", ["fused", "heads_first", "wide"])
def test_strides(layout):
    """Views of a fused q, k, v buffer, heads in front of rows, rows and heads with room between them."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(6)
    lengths, heads, kv, d = [90, 200, 13], 8, 2, 128
    T = sum(lengths)
    if layout == "fused":
        buf = rand(g, (T, (heads + 2 * kv) * d), torch.float16)
        q, k, v = (t.unflatten(1, (-1, d)) for t in buf.split((heads * d, kv * d, kv * d), dim=1))
        out = torch.empty((T, heads, d), dtype=torch.float16, device="cuda")
    elif layout == "heads_first":
        q, k, v = (rand(g, (h, T, d), torch.float16).transpose(0, 1) for h in (heads, kv, kv))
        out = torch.empty((heads, T, d), dtype=torch.float16, device="cuda").transpose(0, 1)
    else:
        q, k, v = (rand(g, (T, h, d + 8), torch.float16)[:, :, :d] for h in (heads, kv, kv))
        out = torch.empty((T, heads, 2 * d), dtype=torch.float16, device="cuda")[:, :, d:]
    ops.attn_prompt(q, k, v, starts_of(lengths), out=out)
    check(out, *reference(q, k, v, spans_of(lengths), d ** -0.5))


@pytest.mark.parametrize("spread,scale", [(30.0, None), (1.0, 3.0), (1e-3, None), (200.0, 1e-4)])
def test_scores_of_all_sizes(spread, scale):
    """Weights that are nearly all on one key, or nearly equal."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(7)
    lengths = [260, 130]
    q, k, v = rand(g, (390, 2, 128), torch.float16, spread), rand(g, (390, 2, 128), torch.float16, spread), rand(g, (390, 2, 128), torch.float16)
    got = ops.attn_prompt(q, k, v, starts_of(lengths), scale=scale)
    check(got, *reference(q, k, v, spans_of(lengths), 128 ** -0.5 if scale is None else scale))


def test_weights_that_grow_along_the_keys():
    """Every key weighs more than all in front of it: the running maximum moves with each tile, up and down again."""
    from rptc_b200 import ops
    T = 900
    q = torch.zeros(T, 1, 128, device="cuda", dtype=torch.float16)
    k = torch.zeros(T, 1, 128, device="cuda", dtype=torch.float16)
    q[:, 0, 0] = 1
    k[:, 0, 0] = torch.cat((torch.arange(600, device="cuda"), torch.arange(300, 0, -1, device="cuda"))) * 0.5
    v = rand(torch.Generator(device="cuda").manual_seed(1), (T, 1, 128), torch.float16)
    got = ops.attn_prompt(q, k, v, starts_of([T]), scale=1.0)
    check(got, *reference(q, k, v, spans_of([T]), 1.0))


def test_one_call_captured_and_replayed_with_other_lengths():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = rand(g, (400, 4, 128), torch.float16), rand(g, (400, 2, 128), torch.float16), rand(g, (400, 2, 128), torch.float16)
    starts = starts_of([400, 0, 0])
    out = torch.zeros_like(q)
    ops.attn_prompt(q, k, v, starts, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_prompt(q, k, v, starts, out=out)
    for lengths in ([400, 0, 0], [1, 398, 1], [130, 130, 140]):
        starts.copy_(starts_of(lengths))
        graph.replay()
        torch.cuda.synchronize()
        check(out, *reference(q, k, v, spans_of(lengths), 128 ** -0.5))


def test_two_streams_at_once():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    sets = [[rand(g, (700, 8, 128), torch.float16) for _ in range(3)] for _ in range(2)]
    lengths = [[700], [100, 350, 250]]
    want = [ops.attn_prompt(*s, starts_of(n)) for s, n in zip(sets, lengths)]
    starts = [starts_of(n) for n in lengths]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attn_prompt(*sets[i], starts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])


def test_indices_outside_the_tensors_are_reported():
    from rptc_b200 import RPTCError, ops
    g = torch.Generator(device="cuda").manual_seed(10)
    q, k, v = (rand(g, (100, 2, 64), torch.float16) for _ in range(3))
    ops.device_status()
    for starts, first, count in (([0, 101], None, None), ([-3, 50], None, None), ([0, 50], [60], [50]), ([0, 50], [0], [-1]), ([50, 20], [0], [10])):
        ops.attn_prompt(q, k, v, int32(starts), *(None if t is None else int32(t) for t in (first, count)))
        with pytest.raises(RPTCError):
            ops.device_status()
    ops.device_status()


def test_many_short_prompts():
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(11)
    lengths = [1 + i * 7 % 23 for i in range(300)]
    T = sum(lengths)
    q, k, v = rand(g, (T, 4, 128), torch.float16), rand(g, (T, 1, 128), torch.float16), rand(g, (T, 1, 128), torch.float16)
    got = ops.attn_prompt(q, k, v, starts_of(lengths))
    check(got, *reference(q, k, v, spans_of(lengths), 128 ** -0.5))


def test_thousands_of_prompts_of_all_lengths():
    """Items of one to many tiles over many more sequences than lanes, some of them empty, in groups whose heads do and do not share an item."""
    from rptc_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(12)
    lengths = [(0, 1, 2, 9, 130, 3, 0, 31)[i % 8] if i % 97 else 300 + i // 3 for i in range(1500)]
    past = [(i * 13) % 40 if i % 5 else 200 * (i % 3) for i in range(1500)]
    T, S = sum(lengths), sum(lengths) + sum(past)
    q, k, v = rand(g, (T, 6, 64), torch.bfloat16), rand(g, (S, 2, 64), torch.bfloat16), rand(g, (S, 2, 64), torch.bfloat16)
    spans = spans_of(lengths, past)
    got = ops.attn_prompt(q, k, v, starts_of(lengths), int32([s[2] for s in spans]), int32([s[3] for s in spans]))
    check(got, *reference(q, k, v, spans, 64 ** -0.5))
    ops.device_status()
