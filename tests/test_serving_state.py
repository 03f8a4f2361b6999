"""What the decode engine refuses leaves its rows as they are: positions, tokens and what the host knows of them."""
import pytest
import torch


def engine(pos, max_pos=16, vocab=50, head_dim=128):
    """An engine's host side on the CPU: its state without weights, and a pass that writes down what it is given."""
    from rptc_b200.llama import LlamaConfig, RPTCLlama
    m = RPTCLlama.__new__(RPTCLlama)
    m.cfg = LlamaConfig(hidden=256, layers=1, heads=2, kv_heads=2, ffn=256, vocab=vocab, max_pos=max_pos, head_dim=head_dim)
    m.rows, m.device, m.kv_bits = len(pos), torch.device("cpu"), 4
    m.pos, m.ids = torch.tensor(pos, dtype=torch.int32), torch.arange(len(pos), dtype=torch.int32)
    m._acc_pool, m.acc_gu2 = torch.ones(3), torch.ones(3)
    m.norm_f = m.head = torch.zeros(1)
    m.sync_positions()
    return m


def state(m):
    return m.pos.tolist(), m.ids.tolist(), m._pos_hi, list(m._behind), m._acc_pool.tolist()


T = lambda *ids: torch.tensor(ids)
BAD = [[T(1)], [T(1), T(2), T(3)], [T(1), T()], [T(1), T(2.0)], [T(1), T(2)[None]], [T(1), T(*range(17))], [T(1), T(50)], [T(-1), T(2)], []]


@pytest.mark.parametrize("bad", BAD, ids=range(len(BAD)))
def test_prompts_that_are_refused_leave_the_rows(bad):
    m = engine([7, 3])
    before = state(m)
    with pytest.raises(ValueError):
        m.prefill_packed(bad)
    assert state(m) == before
    with pytest.raises(ValueError):
        m.extend(bad)
    assert state(m) == before


@pytest.mark.parametrize("tokens", [torch.zeros(2, 17, dtype=torch.long), torch.full((2, 3), 50), torch.zeros(2, 0, dtype=torch.long), torch.zeros(1, 3, dtype=torch.long)])
def test_equal_prompts_that_are_refused_leave_the_rows(tokens):
    m = engine([7, 3])
    before = state(m)
    with pytest.raises(ValueError):
        m.prefill(tokens)
    assert state(m) == before


@pytest.mark.parametrize("bad", [BAD[i] for i in (2, 3, 4, 5, 6, 7)] + [[T(1), T(2), T(3), T(50)], [T(1), T(2), T(*range(17))], [T(1), T(2), T(3), T()]])
def test_texts_that_are_refused_leave_the_rows(bad):
    """All texts are looked at before the first pass, those of later groups too."""
    m = engine([7, 3])
    m._push = lambda *a, **kw: pytest.fail("a pass before all texts were accepted")
    before = state(m)
    with pytest.raises(ValueError):
        m.score(bad)
    assert state(m) == before


@pytest.mark.parametrize("top", [-1, 33, 51])
def test_a_number_of_alternatives_that_is_refused_leaves_the_rows(top):
    m = engine([7, 3])
    m._push = lambda *a, **kw: pytest.fail("a pass before the number was accepted")
    before = state(m)
    with pytest.raises(ValueError):
        m.score([T(1, 2)], top=top)
    assert state(m) == before


def test_a_score_that_ends_early_resets():
    m = engine([7, 3])

    def push(group, whole):
        m.pos.fill_(5)
        m.sync_positions()
        raise MemoryError
    m._push = push
    with pytest.raises(MemoryError):
        m.score([T(1, 2), T(3)])
    assert m.pos.tolist() == [0, 0] and m._pos_hi == 0 and m._behind == [0, 0]


def test_what_is_accepted():
    m = engine([7, 3])
    given = []
    m._push = lambda group, whole: given.append(([p.tolist() for p in group], whole, m.pos.tolist()))
    m._greedy = lambda h: h
    m.extend([T(1, 2, 3, 4, 5, 6, 7, 8, 9), T(49).to(torch.int32)])      # up to max_pos
    m.extend([[1, 2], [3]])
    m.prefill_packed([T(*range(16)), T(0)])
    assert given == [([[1, 2, 3, 4, 5, 6, 7, 8, 9], [49]], False, [7, 3]), ([[1, 2], [3]], False, [7, 3]), ([list(range(16)), [0]], False, [0, 0])]
    m = engine([7, 3])
    with pytest.raises(ValueError):
        m.extend([T(*range(10)), T(1)])                                  # one more than row 0 has room for
    m = engine([0], head_dim=64)
    for call in (m.prefill_packed, m.extend, m.score):
        with pytest.raises(ValueError):
            call([T(1)])
    m = engine([4, 4])
    assert m.score([]) == [] and m.pos.tolist() == [0, 0]


def test_rows_in_front_of_the_first_position_are_not_extended():
    """A token at position -1 belongs to no sequence: it would be left out without a word."""
    m = engine([7, -1])
    m._push = lambda *a, **kw: pytest.fail("a pass behind no position")
    before = state(m)
    with pytest.raises(ValueError):
        m.extend([T(1), T(2, 3)])
    assert state(m) == before
