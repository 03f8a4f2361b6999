"""Log probabilities of given tokens, entropy and largest entries (ops.token_logprobs) against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, targets, top):
    """64 bits, and how far 32 bits may be off: the sums' terms (exp 2^-20 each, with the rounding of its argument) and additions (a chain of n / 256
    and a tree), the roundings of x - max and of the result.  The order of the largest: by value, equal ones by index."""
    x = x.double()
    n = x.shape[1]
    lp = x.log_softmax(-1)
    p = lp.exp()
    apart = torch.where(x == -math.inf, 0.0, x - x.amax(-1, keepdim=True))
    rel = 2.0**-20 + (n / 256 + 32) * 2.0**-24
    spread = (p * apart.abs()).sum(-1)
    entropy = -(torch.where(p > 0, lp, 0.0) * p).sum(-1)
    entropy_tol = 4 * rel * (1 + spread)
    order = x.sort(dim=-1, descending=True, stable=True)
    ids = order.indices[:, :top]
    best = lp.gather(1, ids)
    got = None if targets is None else lp.gather(1, targets.clamp(min=0)[:, None])[:, 0].where(targets >= 0, 0.0)
    tol = lambda at, v: rel + 2.0**-23 * (at.abs().nan_to_num(posinf=0) + v.abs().nan_to_num(posinf=0))
    got_tol = None if targets is None else tol(apart.gather(1, targets.clamp(min=0)[:, None])[:, 0], got)
    return (got, entropy, best, ids), (got_tol, entropy_tol, tol(apart.gather(1, ids), best))


def check(out, want, tol):
    for a, b, t in zip(out[:3], want[:3], tol):
        if b is None:
            assert a is None
            continue
        a = a.double()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        fine = b.isfinite()
        assert ((a - b).abs() <= t)[fine].all(), ((a - b).abs() / t)[fine].max()
    assert torch.equal(out[3], want[3])


def rand(rows, n, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn(rows, n, generator=g, device="cuda")).to(dtype), torch.randint(0, n, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 31, 31), (5, 33, 32), (1, 1000, 5), (4, 1025, 20), (700, 257, 3), (1, 32000, 20), (9, 32001, 1),
                                        (2, 128001, 32), (300, 5000, 0), (1, 160000, 0)])
def test_logprobs(dtype, rows, n, top):
    from rptc_b200 import ops
    x, targets = rand(rows, n, dtype, rows + n)
    out = ops.token_logprobs(x, targets, top)
    check(out, *reference(x, targets, top))
    again = ops.token_logprobs(x, targets, top)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    alone = ops.token_logprobs(x, None, top)
    assert alone[0] is None and all(torch.equal(a, b) for a, b in zip(out[1:], alone[1:]))
    ops.device_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,skip", [(1000, 1), (1003, 0), (4099, 3), (33, 7)])
def test_rows_off_every_boundary(dtype, n, skip):
    """A view whose rows start anywhere; what lies between them is not read."""
    from rptc_b200 import ops
    wide = torch.full((6, n + 13), math.nan, dtype=dtype, device="cuda")
    x, targets = rand(6, n, dtype, n)
    wide[:, skip:skip + n] = x
    check(ops.token_logprobs(wide[:, skip:skip + n], targets, 7), *reference(x, targets, 7))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [50, 3000, 40000])
def test_forbidden_tokens(dtype, n):
    """-inf, and the type's lowest value, on nearly everything; a row with one token left, and one with none."""
    from rptc_b200 import ops
    x, targets = rand(6, n, dtype, n)
    g = torch.Generator(device="cuda").manual_seed(1)
    x[0].masked_fill_(torch.rand(n, generator=g, device="cuda") < 0.9, -math.inf)
    x[1].masked_fill_(torch.rand(n, generator=g, device="cuda") < 0.9, torch.finfo(dtype).min)
    x[2] = -math.inf
    x[2, n // 2] = 1.0
    x[3] = -math.inf
    x[4, : n - 3] = -math.inf
    out = ops.token_logprobs(x, targets, 5)
    want, tol = reference(x, targets, 5)
    assert out[0][3].isnan() and out[1][3].isnan() and out[2][3].isnan().all() and out[3][3].tolist() == [0, 1, 2, 3, 4]
    keep = [0, 1, 2, 4, 5]
    check([t[keep] for t in out], [t[keep] for t in want], [t[keep] for t in tol])
    assert out[1][2] == 0 and out[2][2, 0] == 0 and out[3][2, 0] == n // 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("n", [40, 5000, 50000])
def test_ties_go_to_the_lowest_index(dtype, n):
    from rptc_b200 import ops
    x = torch.zeros(4, n, dtype=dtype, device="cuda")
    x[0, ::2] = -0.0                                          # equal to 0
    x[1] = (torch.arange(n, device="cuda") % 7 == 3).to(dtype)
    x[2, n // 3:] = 2.0
    x[3] = torch.arange(n, device="cuda").flip(0).clamp(max=11).to(dtype)
    targets = torch.tensor([0, 3, n - 1, n // 2], device="cuda")
    check(ops.token_logprobs(x, targets, 32), *reference(x, targets, 32))


@pytest.mark.parametrize("n", [300, 30000])
def test_large_and_close_values(n):
    """Far from zero, where x - max is what counts; one entry far above all others; everything in one thread's reach."""
    from rptc_b200 import ops
    x, targets = rand(5, n, torch.float32, 5)
    x[0] += 1000
    x[1] -= 3e4
    x[2, 17] = 500
    x[3] = 1e30 * x[3]
    x[4, :40] += 50                                           # all of the largest side by side
    check(ops.token_logprobs(x, targets, 32), *reference(x, targets, 32))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,top", [(3, 32000, 20), (400, 32000, 32), (400, 128001, 20)])
def test_largest_entries_side_by_side(dtype, rows, n, top):
    """The largest lie apart by lengths that the kernel's strides divide, or next to one another, or all but one are -inf."""
    from rptc_b200 import ops
    x, targets = rand(rows, n, dtype, 7 * rows + n)
    for r in range(rows):
        step = (1, 4, 8, 1024, 2048, 4096, 8192, 1000)[r % 8]
        at = torch.arange(r, n, step, device="cuda")[:top + 3]
        x[r, at] = 20 + torch.arange(len(at), device="cuda", dtype=dtype) / 8
    x[0] = -math.inf
    x[0, n // 3] = 1
    targets[0] = n // 3
    if rows > 8:
        x[8, n // 2:] = -math.inf
        x[9, 5] = x[9, 4096 + 5] = math.inf
    out = ops.token_logprobs(x, targets, top)
    want, tol = reference(x, targets, top)
    if rows > 8:      # a row with +inf has no probabilities
        assert out[0][9].isnan() and out[1][9].isnan() and out[2][9].isnan().all()
    keep = torch.arange(rows, device="cuda") != 9
    check([o[keep] for o in out], [w[keep] for w in want], [t[keep] for t in tol])
    ops.device_status()


def test_rows_without_numbers():
    from rptc_b200 import ops
    x, targets = rand(4, 2000, torch.float32, 6)
    x[0, 1999] = math.nan
    x[2, 0] = math.inf
    clean = ops.token_logprobs(x[1::2].contiguous(), targets[1::2].contiguous(), 4)
    out = ops.token_logprobs(x, targets, 4)
    for r in (0, 2):
        assert out[0][r].isnan() and out[1][r].isnan() and out[2][r].isnan().all()
        assert len(set(out[3][r].tolist())) == 4 and ((out[3][r] >= 0) & (out[3][r] < 2000)).all()
    assert all(torch.equal(a[1::2], b) for a, b in zip(out, clean))


def test_targets_of_no_token_and_outside():
    from rptc_b200 import RPTCError, ops
    x, targets = rand(4, 500, torch.float16, 7)
    want = ops.token_logprobs(x, targets)[0]
    ops.device_status()
    targets[1] = -1
    got = ops.token_logprobs(x, targets)[0]
    ops.device_status()
    assert got[1] == 0 and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
    for bad in (-2, 500, 2**40):
        targets[2] = bad
        got = ops.token_logprobs(x, targets)[0]
        with pytest.raises(RPTCError):
            ops.device_status()
        assert got[2].isnan() and torch.equal(got[[0, 3]], want[[0, 3]])


def test_captured_and_on_two_streams():
    from rptc_b200 import ops
    for rows in (1, 300):
        x, targets = rand(rows, 40000, torch.float16, 8)
        other, _ = rand(rows, 40000, torch.float16, 9)
        want = [ops.token_logprobs(t, targets, 6) for t in (x, other)]
        graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
        for t, s in zip((x, other), streams):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = ops.token_logprobs(t, targets, 6)
            graphs.append((graph, out))
        for _ in range(5):
            for (graph, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
