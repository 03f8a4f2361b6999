"""The decode engine with prompts of different lengths, continued conversations, a 4-bit KV cache and scores, against fp32 torch forwards
of the same network.  Tolerance as for the engine's other paths: 1e-2 of the largest logit of a position."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(rows=3, kv_heads=2, kv_bits=16, max_pos=96, incoherent=True, hidden=512, seed=7, heads=4):
    from rptc_b200.llama import LlamaConfig, RPTCLlama
    cfg = LlamaConfig(hidden=hidden, layers=2, heads=heads, kv_heads=kv_heads, ffn=1024, vocab=1024, max_pos=max_pos, weight_scale=0.05 if hidden < 4096 else 0.02)
    return RPTCLlama(cfg, rows=rows, seed=seed, incoherent=incoherent, kv_bits=kv_bits)


def texts(lengths, vocab=1024, seed=11):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, vocab, (n,), device="cuda", generator=g) for n in lengths]


def reference(model, tokens, own=0, bits=16, row=None):
    """fp32 logits [T, vocab] of one row; with bits = 4 the first `own` queries see each other's keys and values as they are, all others what the row's cache
    holds.  (Codes of this forward's own keys would not do: a thousandth of a difference moves one in some hundred values across a border, by a whole step.)  What
    the cache holds is checked on the way: half a step off the keys and values, and what the activations differ by."""
    from rptc_b200 import ops
    cfg, T = model.cfg, len(tokens)
    h = model.embed[tokens].float()[None]
    half = cfg.head_dim // 2
    ang = torch.arange(T, device="cuda", dtype=torch.float32)[:, None] * cfg.rope_theta ** (-torch.arange(half, device="cuda", dtype=torch.float32) * 2 / cfg.head_dim)
    cs, sn = ang.cos()[None, :, None], ang.sin()[None, :, None]
    rms = lambda x, w: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.rms_eps) * w.float()

    def rope(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cs - b * sn, b * cs + a * sn), -1)

    q_dim, kv_dim, rep = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim, cfg.heads // cfg.kv_heads
    mask = torch.full((T, T), -math.inf, device="cuda").triu(1)
    for layer, b in enumerate(model.blocks):
        qkv = rms(h, b.norm1) @ b.qkv.effective_weight().t()
        q, k, v = qkv.split((q_dim, kv_dim, kv_dim), -1)
        q, k, v = rope(q.unflatten(2, (-1, 128))), rope(k.unflatten(2, (-1, 128))), v.unflatten(2, (-1, 128))

        def attention(k, v):
            p = torch.einsum("bthd,bshd->bhts", q, k.repeat_interleave(rep, 2)) * cfg.head_dim ** -0.5 + mask
            return torch.einsum("bhts,bshd->bthd", p.softmax(-1), v.repeat_interleave(rep, 2)).reshape(1, T, q_dim)

        if bits == 4:
            held = [t[row, :T].float()[None] for t in ops.kv4_values(model.kv4[layer], torch.full((model.rows,), T, dtype=torch.int32, device="cuda"))]
            for is_, was in zip(held, (k, v)):
                g = was.unflatten(-1, (4, 32))
                step = (g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) / 15
                assert ((is_.unflatten(-1, (4, 32)) - g).abs() <= 0.51 * step + 2e-2 * was.abs().max()).all()
            cached = attention(*held)
            o = torch.cat((attention(k, v)[:, :own], cached[:, own:]), 1)
        else:
            o = attention(k, v)
        h = h + o @ b.o.effective_weight().t()
        gu = rms(h, b.norm2) @ b.gate_up.effective_weight().t()
        h = h + (torch.nn.functional.silu(gu[..., : cfg.ffn]) * gu[..., cfg.ffn:]) @ b.down.effective_weight().t()
    return (rms(h, model.norm_f) @ model.head.float().t())[0]


def close(got, want, tol=1e-2):
    err = ((got.float() - want).abs().max() / want.abs().max()).item()
    print("err %.2e" % err)
    assert err <= tol, err


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("incoherent,kv_heads", [(True, 2), (True, 4), (False, 2)])
@pytest.mark.parametrize("lengths", [[40, 1, 17], [1, 1, 1], [2, 3, 3]])
def test_prompts_of_different_lengths_then_decoding(kv_bits, incoherent, kv_heads, lengths):
    model = make(kv_heads=kv_heads, kv_bits=kv_bits, incoherent=incoherent)
    prompts = texts(lengths)
    logits = model.prefill_packed(prompts).clone()
    whole = [p.tolist() for p in prompts]
    assert model.pos.tolist() == lengths
    for r, p in enumerate(prompts):
        close(logits[r], reference(model, p, len(p), kv_bits, r)[-1])
    for use_graph in (False, True):
        if use_graph:
            model.capture()
        for _ in range(3):
            for r in range(3):
                whole[r].append(model.ids[r].item())
            model.step()
            for r in range(3):
                close(model.logits[r], reference(model, torch.tensor(whole[r], device="cuda"), lengths[r], kv_bits, r)[-1])
    from rptc_b200 import ops
    ops.device_status()


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_conversations_go_on(kv_bits):
    model = make(kv_bits=kv_bits, max_pos=128)
    first, second = texts([20, 3, 31]), texts([5, 40, 1], seed=5)
    model.prefill_packed(first)
    said = [[t.item()] for t in model.ids]
    model.step()
    logits = model.extend([torch.cat((torch.tensor(s, device="cuda")[1:], p)) if len(s) > 1 else p for s, p in zip(said, second)])
    for r in range(3):
        tokens = torch.cat((first[r], torch.tensor(said[r], device="cuda"), second[r]))
        assert model.pos[r].item() == len(tokens)
        close(logits[r], reference(model, tokens, len(first[r]), kv_bits, r)[-1])
    whole = [torch.cat((first[r], torch.tensor(said[r] + [model.ids[r].item()], device="cuda")[:1], second[r], model.ids[r:r + 1].long())) for r in range(3)]
    model.step()
    for r in range(3):
        close(model.logits[r], reference(model, whole[r], len(first[r]), kv_bits, r)[-1])


def test_equal_prompts_agree_with_prefill():
    """The packed pass and the one for equal lengths give the same caches, but for the rounding of rotated keys' last bits, and the same logits."""
    a, b = make(rows=2), make(rows=2)
    tokens = torch.stack(texts([33, 33]))
    la, lb = a.prefill(tokens).clone(), b.prefill_packed(list(tokens))
    close(lb, la.float(), 5e-3)
    for x, y in zip(a.kcache + a.vcache, b.kcache + b.vcache):
        close(y[:, :33], x[:, :33].float(), 5e-3)
    assert not any(x[:, 33:].any() for x in b.kcache)


def test_four_bits_take_prefill_and_a_third_of_the_memory():
    model = make(kv_bits=4, rows=2)
    tokens = torch.stack(texts([25, 25]))
    logits = model.prefill(tokens)
    for r in range(2):
        close(logits[r], reference(model, tokens[r], 25, 4, r)[-1])
    wide = make(kv_bits=16, rows=2)
    assert model.bytes_per_token(100)["kv"] * 512 == wide.bytes_per_token(100)["kv"] * 160
    assert sum(t.numel() * t.element_size() for t in model.kv4[0]) * 512 == 160 * sum(t.numel() * t.element_size() for t in (wide.kcache[0], wide.vcache[0]))


@pytest.mark.parametrize("hidden,kv_heads,rows,max_pos", [(4096, 8, 1, 64), (4096, 32, 2, 64), (768, 2, 2, 64), (512, 2, 2, 1500)])
def test_four_bits_in_every_chain(hidden, kv_heads, rows, max_pos):
    """The short chains of hidden 4096, the unfused one, and a cache so long that its attention takes two launches."""
    model = make(rows=rows, kv_heads=kv_heads, kv_bits=4, hidden=hidden, max_pos=max_pos, heads=hidden // 128)
    tokens = torch.stack(texts([6] * rows))
    for use_graph in (False, True):
        model.reset()
        if use_graph:
            model.capture()
        for t in range(6):
            model.ids.copy_(tokens[:, t].to(torch.int32))
            model.step()
            for r in range(rows):
                close(model.logits[r], reference(model, tokens[r, :t + 1], 0, 4, r)[-1], 1e-2 if hidden < 4096 else 2e-2)


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_rows_fill_their_caches_by_themselves(kv_bits):
    """A row has the room behind its own position, wherever the others are."""
    model = make(rows=2, kv_bits=kv_bits)
    first, second = texts([90, 2]), texts([1, 60], seed=3)
    model.prefill_packed(first)
    logits = model.extend(second)
    for r in range(2):
        tokens = torch.cat((first[r], second[r]))
        close(logits[r], reference(model, tokens, len(first[r]), kv_bits, r)[-1])
    assert model.pos.tolist() == [91, 62] and model._pos_hi == 91 and model._behind == [0, 29]
    for _ in range(5):
        model.step()
    with pytest.raises(RuntimeError):
        model.step()
    with pytest.raises(ValueError):
        model.extend(texts([1, 1]))
    model.pos.copy_(torch.tensor([10, 80], device="cuda"))
    model.sync_positions()
    with pytest.raises(ValueError):
        model.extend(texts([1, 17]))
    model.extend(texts([86, 16]))
    assert model.pos.tolist() == [96, 96]


def test_launches_of_long_four_bit_caches():
    """A second launch where a workspace takes the parts of a row."""
    import ctypes

    from rptc_b200 import ops
    from rptc_b200._lib import lib
    for rows, max_pos in ((1, 1024), (1, 2048), (64, 2048), (64, 2049)):
        cache = ops.kv4_cache(rows, max_pos, 2)
        joins = ops.attn_decode_kv4_joins(cache, 4)
        assert joins == (lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(ops._kv_cache(cache, cache[0].device)), 4) > 0)
        assert joins == (max_pos > 2048 or (rows, max_pos) == (1, 2048))
    long, short = make(rows=2, kv_bits=4, max_pos=1500), make(rows=2, kv_bits=4)
    for model in (long, short):
        model.step()
    assert long.launches_per_step == short.launches_per_step + len(long.blocks)


def test_scores_are_the_log_probabilities_of_the_next_tokens():
    model = make(rows=2)
    prompts = texts([30, 1, 9, 2, 50])
    found = model.score(prompts, top=3)
    assert len(found) == 5 and model.pos.tolist() == [0, 0]
    for p, (logprob, entropy, top, ids) in zip(prompts, found):
        assert logprob.shape == entropy.shape == (len(p) - 1,) and top.shape == ids.shape == (len(p) - 1, 3)
        if len(p) == 1:
            continue
        want = reference(model, p)[:-1].log_softmax(-1)
        room = 2e-2 * reference(model, p).abs().max().item()       # a logit and the sum over all are each off by at most 1e-2 of the largest
        assert ((logprob - want.gather(1, p[1:, None])[:, 0]).abs() <= room).all()
        assert ((top - want.gather(1, ids)).abs() <= room).all() and (top[:, :-1] >= top[:, 1:]).all()
        assert ((entropy + (want.exp() * want).sum(-1)).abs() <= 4 * room).all()


def test_what_is_refused():
    from rptc_b200.llama import LlamaConfig, RPTCLlama
    model = make(rows=2)
    a, b = texts([5, 6])
    for bad in ([a], [a, b, a], [a, b[:0]], [a, b.float()], [a, b[None]]):
        with pytest.raises(ValueError):
            model.prefill_packed(bad)
    with pytest.raises(ValueError):
        model.prefill_packed([a, texts([97])[0]])
    for bad in (-1, 1024):                                           # no such token
        with pytest.raises(ValueError):
            model.prefill_packed([a, torch.tensor([3, bad])])
        with pytest.raises(ValueError):
            model.score([torch.tensor([bad, 2])])
    model.prefill_packed(texts([90, 1]))
    with pytest.raises(ValueError):
        model.extend([texts([7])[0], a])
    with pytest.raises(ValueError):
        RPTCLlama(LlamaConfig(hidden=512, layers=1, heads=8, kv_heads=8, head_dim=64, ffn=1024, vocab=64), kv_bits=4)
    with pytest.raises(ValueError):
        RPTCLlama(LlamaConfig(hidden=512, layers=1, heads=4, kv_heads=4, ffn=1024, vocab=64), kv_bits=8)
