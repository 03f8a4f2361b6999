"""What the serving operators' front end refuses on the GPU, before anything is launched."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16, device="cuda")


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prompt(**change):
    from rptc_b200 import ops
    a = dict(q=half(6, 4, 128), k=half(6, 2, 128), v=half(6, 2, 128), starts=i32(0, 4, 6))
    a.update(change)
    return ops.attn_prompt(**a)


def append(**change):
    from rptc_b200 import ops
    a = dict(x=half(3, 8 * 128), pos=i32(0, 1, 2), angles=torch.zeros(16, 64, 2, device="cuda"), cache=ops.kv4_cache(3, 16, 2), heads=4, kv_heads=2)
    a.update(change)
    return ops.qkv_append(**a)


def decode(**change):
    from rptc_b200 import ops
    a = dict(q=half(3, 4 * 128), pos=i32(0, 1, 2), cache=ops.kv4_cache(3, 16, 2), heads=4)
    a.update(change)
    return ops.attn_decode_kv4(**a)


def values(**change):
    from rptc_b200 import ops
    a = dict(cache=ops.kv4_cache(3, 16, 2), count=i32(0, 1, 2))
    a.update(change)
    return ops.kv4_values(**a)


def logprobs(**change):
    from rptc_b200 import ops
    a = dict(logits=half(3, 50), targets=torch.zeros(3, dtype=torch.int64, device="cuda"), top=2)
    a.update(change)
    return ops.token_logprobs(**a)


def bad_calls():
    return [
        (prompt, [dict(q=half(6, 4, 128).float()), dict(k=half(6, 2, 128).bfloat16()), dict(v=half(5, 2, 128)), dict(k=half(6, 2, 64), v=half(6, 2, 64)), dict(q=half(6, 3, 128)),
                  dict(q=half(6, 4, 96), k=half(6, 2, 96), v=half(6, 2, 96)), dict(q=half(6, 512)), dict(q=half(6, 4, 128).cpu()), dict(starts=i32(0, 4, 6).long()), dict(starts=i32(0, 4, 6).cpu()),
                  dict(starts=i32(0, 4, 6)[:0]), dict(kv_first=i32(0, 0)), dict(kv_first=i32(0, 0), kv_len=i32(1)), dict(k=half(5, 2, 128), v=half(5, 2, 128)), dict(out=half(6, 4, 64)),
                  dict(out=half(6, 4, 128).float()), dict(q=half(6, 4, 256)[..., ::2]), dict(q=half(6 * 512 + 8)[1:6 * 512 + 1].view(6, 4, 128)), dict(q=half(6, 4, 130)[..., :128]),
                  dict(k=half(1, 2, 128).expand(6, 2, 128)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)]),
        (append, [dict(x=half(3, 8 * 128).bfloat16()), dict(x=half(3, 7 * 128)), dict(x=half(8 * 128)), dict(x=half(3, 16 * 128)[:, ::2]), dict(x=half(1, 8 * 128).expand(3, -1)), dict(pos=i32(0, 1, 2).long()),
                  dict(pos=i32(0, 1)), dict(angles=torch.zeros(15, 64, 2, device="cuda")), dict(angles=half(16, 64, 2)), dict(cache=(half(3, 16, 2, 64),) * 2), dict(cache=(half(3, 16, 2, 128),) * 3),
                  dict(heads=3), dict(heads=0), dict(kv_heads=4), dict(slots=i32(0, 1)), dict(slots=i32(0, 1, 2).long()), dict(signs_out=half(8 * 128)), dict(signs_out=half(64), transform=True),
                  dict(clear=True), dict(out=half(3, 3 * 128)), dict(out=half(2, 8 * 128)), dict(out=half(3, 8 * 128).float()), dict(out=half(3, 8 * 128 + 1)[:, 1:])]),
        (decode, [dict(q=half(3, 4 * 128).float()), dict(q=half(2, 4 * 128)), dict(q=half(3, 3 * 128)), dict(q=half(3, 4 * 128 + 1)[:, 1:]), dict(pos=i32(0, 1)), dict(pos=i32(0, 1, 2).long()),
                  dict(cache=(half(3, 16, 2, 128), half(3, 16, 2, 128))), dict(heads=3), dict(heads=0), dict(heads=-2), dict(heads=5000, q=half(3, 5000 * 128)), dict(out=half(3, 3 * 128)),
                  dict(out=half(3, 4 * 128).float()), dict(scale=0.0), dict(scale=math.nan), dict(signs_in=half(128)), dict(signs_in=half(4 * 128).float())]),
        (values, [dict(cache=(half(3, 16, 2, 128), half(3, 16, 2, 128))), dict(count=i32(0, 1)), dict(count=i32(0, 1, 2).long()), dict(out=(half(3, 16, 2, 64), half(3, 16, 2, 128))),
                  dict(out=(half(3, 16, 2, 128), half(3, 16, 2, 128).float()))]),
        (logprobs, [dict(logits=half(3, 50).long()), dict(logits=half(50)), dict(logits=half(3, 0)), dict(logits=half(3, 100)[:, ::2]), dict(logits=half(1, 50).expand(3, -1)), dict(logits=half(3, 50).cpu()),
                    dict(targets=i32(0, 1, 2)), dict(targets=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(targets=torch.zeros(3, dtype=torch.int64)), dict(top=-1), dict(top=33), dict(top=51)]),
    ]


@pytest.mark.parametrize("call", [prompt, append, decode, values, logprobs])
def test_refused(call):
    from rptc_b200 import ops
    call()
    torch.cuda.synchronize()
    ops.device_status()
    for change in dict(bad_calls())[call]:
        with pytest.raises(RuntimeError):
            call(**change)
    torch.cuda.synchronize()
    ops.device_status()


def test_nothing_to_do():
    """Calls without rows or tokens answer with empty results."""
    from rptc_b200 import ops
    assert prompt(q=half(0, 4, 128), starts=i32(0), k=half(0, 2, 128), v=half(0, 2, 128)).shape == (0, 4, 128)
    assert append(x=half(0, 8 * 128), pos=i32()).shape == (0, 8 * 128)
    for t in logprobs(logits=half(0, 50), targets=torch.zeros(0, dtype=torch.int64, device="cuda")):
        assert t.shape[0] == 0
    out = torch.full((6, 4, 128), 3.0, dtype=torch.float16, device="cuda")
    assert (prompt(starts=i32(0), out=out) == 3).all()         # rows of no sequence
    ops.device_status()
