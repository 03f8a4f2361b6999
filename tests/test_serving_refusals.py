"""What the serving operators refuse, before anything reaches a GPU: their arguments at the C boundary and at the tensor front end."""
import ctypes

import pytest
import torch

BASE, UNALIGNED = 1 << 12, (1 << 12) + 8


@pytest.fixture(autouse=True)
def made_up_addresses_stay_off_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses stay off a GPU")


def cache(**kw):
    from rptc_b200._lib import KVCache
    return KVCache(**{**dict(k=BASE, k_scales=BASE, v=BASE, v_scales=BASE, rows=2, max_pos=16, kv_heads=2, bits=4), **kw})


def prompt(**kw):
    from rptc_b200 import lib
    from rptc_b200._lib import PromptAttention
    a = dict(q=BASE, k=BASE, v=BASE, out=BASE, starts=BASE, kv_first=None, kv_len=None, tokens=8, kv_tokens=8, sequences=1, q_row=512, q_head=128, k_row=256,
             k_head=128, v_row=256, v_head=128, out_row=512, out_head=128, heads=4, kv_heads=2, d=128, dtype=0, scale=0.1)
    return lib().rptc_attn_prompt(ctypes.byref(PromptAttention(**{**a, **kw})), None)


def append(c=None, **kw):
    from rptc_b200 import lib
    from rptc_b200._lib import Append
    a = dict(x=BASE, ld_x=1024, signs_out=None, slots=None, pos=BASE, angles=BASE, out=BASE, ld_out=1024, tokens=2, heads=4, x_is_f32=0, clear=0, transform=1, out_kv=1,
             scale=1.0, cache=c or cache())
    return lib().rptc_qkv_append(ctypes.byref(Append(**{**a, **kw})), None)


def decode(c=None, **kw):
    from rptc_b200 import lib
    a = {**dict(q=BASE, ld_q=512, pos=BASE, out=BASE, ld_out=512, heads=4, scale=0.1, signs=None, ws=None, ws_bytes=0), **kw}
    return lib().rptc_attn_decode_kv4(a["q"], a["ld_q"], a["pos"], ctypes.byref(c or cache()), a["out"], a["ld_out"], a["heads"], a["scale"], a["signs"], a["ws"],
                                      a["ws_bytes"], None)


def logprobs(**kw):
    from rptc_b200 import lib
    a = {**dict(logits=BASE, dtype=0, ld=100, targets=BASE, logprob=BASE, entropy=BASE, top_lp=BASE, top_ids=BASE, rows=3, n=100, top=5), **kw}
    return lib().rptc_token_logprobs(a["logits"], a["dtype"], a["ld"], a["targets"], a["logprob"], a["entropy"], a["top_lp"], a["top_ids"], a["rows"], a["n"], a["top"], None)


NO_DEVICE = (-5, -8)      # what a call that nothing is wrong with gets without a GPU


@pytest.mark.parametrize("status,kw", [
    (-1, dict(q=None)), (-1, dict(out=None)), (-1, dict(starts=None)), (-1, dict(kv_first=BASE)), (-1, dict(kv_len=BASE)), (-1, dict(dtype=2)), (-1, dict(scale=0.0)),
    (-1, dict(scale=-1.0)), (-1, dict(scale=float("nan"))), (-1, dict(scale=float("inf"))), (-4, dict(d=96)), (-4, dict(d=256)), (-2, dict(heads=3)), (-2, dict(heads=0)),
    (-2, dict(tokens=-1)), (-2, dict(kv_tokens=9)), (-2, dict(q_head=64)), (-2, dict(k_row=0)), (-3, dict(v_row=260)), (-3, dict(q=UNALIGNED)), (-3, dict(out=BASE + 2)),
    (-7, dict(sequences=65536)), (-7, dict(tokens=(1 << 24) + 1, kv_tokens=(1 << 24) + 1)), (-7, dict(heads=8192, kv_heads=8192))])
def test_prompt_attention_refuses(status, kw):
    assert prompt(**kw) == status


@pytest.mark.parametrize("status,kw", [
    (-1, dict(x=None)), (-1, dict(pos=None)), (-1, dict(angles=None)), (-1, dict(out=None)), (-1, dict(signs_out=BASE, transform=0)), (-1, dict(clear=1)),
    (-2, dict(heads=3)), (-2, dict(heads=0)), (-2, dict(ld_x=1016)), (-2, dict(ld_out=1016)), (-2, dict(ld_out=504, out_kv=0)), (-2, dict(tokens=3)), (-2, dict(tokens=-1)),
    (-3, dict(x=UNALIGNED)), (-3, dict(out=UNALIGNED)), (-3, dict(signs_out=UNALIGNED)), (-3, dict(angles=UNALIGNED)), (-3, dict(ld_x=1028)), (-3, dict(ld_out=1028)),
    (-7, dict(tokens=(1 << 24) + 1, slots=BASE)), (-7, dict(heads=8192, ld_x=1 << 24, ld_out=1 << 24))])
def test_append_refuses(status, kw):
    assert append(**kw) == status


CACHES = [(-1, dict(k=None)), (-1, dict(v_scales=None)), (-1, dict(bits=8)), (-2, dict(rows=0)), (-2, dict(max_pos=0)), (-2, dict(kv_heads=-1)), (-3, dict(k=UNALIGNED)),
          (-3, dict(k_scales=UNALIGNED)), (-7, dict(rows=65536)), (-7, dict(max_pos=(1 << 24) + 1)), (-7, dict(kv_heads=4097))]


@pytest.mark.parametrize("status,kw", CACHES)
def test_caches_that_are_none(status, kw):
    from rptc_b200 import lib
    bad = cache(**kw)
    assert append(bad) == status and decode(bad) == status
    assert lib().rptc_kv4_values(ctypes.byref(bad), BASE, BASE, BASE, None) == status
    assert lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(bad), 4) == 0


@pytest.mark.parametrize("status,kw", [
    (-1, dict(q=None)), (-1, dict(pos=None)), (-1, dict(out=None)), (-1, dict(scale=0.0)), (-1, dict(scale=float("nan"))), (-2, dict(heads=3)), (-2, dict(heads=0)),
    (-2, dict(ld_q=504)), (-2, dict(ld_out=504)), (-3, dict(q=UNALIGNED)), (-3, dict(out=UNALIGNED)), (-3, dict(signs=UNALIGNED)), (-3, dict(ld_q=516)), (-3, dict(ld_out=516)),
    (-7, dict(heads=8192, ld_q=1 << 24, ld_out=1 << 24))])
def test_decode_refuses(status, kw):
    assert decode(**kw) == status


def test_decode_wants_its_workspace():
    from rptc_b200 import lib
    long = cache(max_pos=100000)
    need = lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(long), 4)
    assert need > 0 and need % 8 == 0
    assert decode(long) == -1 and decode(long, ws=BASE, ws_bytes=need - 1) == -1 and decode(long, ws=BASE + 16, ws_bytes=need) == -3
    assert decode(cache(bits=16, k_scales=None, v_scales=None)) == -4


@pytest.mark.parametrize("status,kw", [
    (-1, dict(logits=None)), (-1, dict(dtype=3)), (-1, dict(dtype=-1)), (-1, dict(logprob=None)), (-1, dict(top_ids=None)), (-1, dict(top_lp=None)), (-1, dict(top=-1)),
    (-2, dict(n=0)), (-2, dict(rows=-1)), (-2, dict(ld=99)), (-2, dict(n=4, ld=4)), (-3, dict(logits=BASE + 1)), (-3, dict(logits=BASE + 2, dtype=2)), (-7, dict(top=33)),
    (-7, dict(n=(1 << 24) + 1, ld=1 << 25)), (-7, dict(rows=(1 << 24) + 1))])
def test_logprobs_refuse(status, kw):
    assert logprobs(**kw) == status


def test_calls_that_nothing_is_wrong_with_get_as_far_as_the_device():
    assert prompt() in NO_DEVICE and prompt(kv_first=BASE, kv_len=BASE, kv_tokens=100) in NO_DEVICE and append() in NO_DEVICE and decode() in NO_DEVICE
    assert logprobs() in NO_DEVICE and logprobs(targets=None, logprob=None, top=0, top_lp=None, top_ids=None) in NO_DEVICE
    assert append(cache(bits=16, k_scales=None, v_scales=None)) in NO_DEVICE


def test_front_end_refuses_what_is_not_on_a_gpu():
    from rptc_b200 import ops
    h, i = torch.float16, torch.int32
    q = torch.zeros(4, 2, 128, dtype=h)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_prompt(q, q, q, torch.zeros(2, dtype=i))
    c = ops.kv4_cache(2, 8, 1, device="cpu")
    x = torch.zeros(2, 3 * 128, dtype=h)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qkv_append(x, torch.zeros(2, dtype=i), torch.zeros(8, 64, 2), c, 1, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_kv4(x, torch.zeros(2, dtype=i), c, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv4_values(c, torch.zeros(2, dtype=i))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.token_logprobs(torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="cache"):
        ops.attn_decode_kv4(x, torch.zeros(2, dtype=i), c[:3], 3)
