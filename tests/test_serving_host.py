"""What the serving operators refuse, on the host alone: nothing is launched."""
import ctypes as C

import pytest
import torch

from metalhlo_amd import _lib, kernels
from tests.paged_util import scale_byte

BF16, F16, F32, I32, I64 = 3, 0, 1, 7, 8


class Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("keys", "values", "key_scales", "value_scales")] + [(n, C.c_int64) for n in ("pages", "heads", "page_size", "head_size")]


class Sequences(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("table", "lengths", "starts")] + [(n, C.c_int64) for n in ("sequences", "width", "tokens")]


P = 1 << 20                                    # an aligned address that nothing is read from: every call here ends before a launch


def cache(**kw):
    return Cache(**{**dict(keys=P, values=P, key_scales=None, value_scales=None, pages=4, heads=2, page_size=16, head_size=64), **kw})


def seqs(**kw):
    return Sequences(**{**dict(table=P, lengths=P, starts=P, sequences=2, width=2, tokens=3), **kw})


def append(c, s, k=P, v=P, q=None, q_out=None, heads=0, freqs=None, positions=0, rotated=0, strides=(128, 64) * 4, dtype=BF16):
    st = (C.c_int64 * 8)(*strides) if strides else None
    return _lib.load().mhip_paged_append(None, C.byref(c) if c else None, C.byref(s) if s else None, k, v, q, q_out, heads, freqs, positions, rotated, st, dtype)


def attend(c, s, q=P, o=P, heads=4, strides=(256, 64) * 2, dtype=BF16, work=None, size=0):
    st = (C.c_int64 * 4)(*strides) if strides else None
    return _lib.load().mhip_paged_attention(None, C.byref(c) if c else None, C.byref(s) if s else None, q, o, heads, 1.0, 1, st, dtype, work, size)


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("change,code", [
    (dict(pages=0), 1), (dict(pages=-1), 1), (dict(heads=0), 1), (dict(heads=2000), 2), (dict(keys=None), 1), (dict(values=None), 1), (dict(key_scales=P), 1),
    (dict(value_scales=P), 1), (dict(head_size=48), 2), (dict(head_size=160), 2), (dict(head_size=0), 2), (dict(page_size=8), 2), (dict(page_size=48), 2), (dict(page_size=512), 2),
    (dict(keys=P + 8), 2), (dict(values=P + 2), 2)], ids=str)
def test_caches_that_are_none(call, change, code):
    assert call(cache(**change), seqs()) == code, _lib.load().mhip_last_error()


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("change,code", [
    (dict(sequences=-1), 1), (dict(width=-1), 1), (dict(tokens=-1), 1), (dict(starts=None), 1), (dict(lengths=None), 1), (dict(table=None), 1),
    (dict(sequences=70000), 2), (dict(width=1 << 21), 2), (dict(tokens=1 << 25), 2)], ids=str)
def test_sequences_that_are_none(call, change, code):
    assert call(cache(), seqs(**change)) == code, _lib.load().mhip_last_error()


@pytest.mark.parametrize("call", [append, attend])
def test_nothing_to_do(call):
    assert call(cache(), seqs(tokens=0)) == 0 and call(cache(), seqs(sequences=0)) == 0
    assert call(None, seqs()) == 1 and call(cache(), None) == 1
    assert call(cache(), seqs(), dtype=F32) == 2 and b"dtype" in _lib.load().mhip_last_error()


def test_append_refuses():
    c, s = cache(), seqs()
    assert append(c, s, k=None) == 1 and append(c, s, v=None) == 1 and append(c, s, strides=None) == 1
    assert append(c, s, k=P + 2) == 2 and append(c, s, strides=(130, 64) * 4) == 2
    assert append(c, s, rotated=16) == 1                                  # no freqs
    assert append(c, s, freqs=P, positions=4, rotated=24) == 2 and append(c, s, freqs=P, positions=4, rotated=80) == 2 and append(c, s, freqs=P, positions=4, rotated=-16) == 2
    assert append(c, s, freqs=P, positions=-1, rotated=16) == 1 and append(c, s, freqs=P + 4, positions=4, rotated=16) == 2
    assert append(c, s, q=P, heads=4, freqs=P, positions=4, rotated=16) == 1 and append(c, s, q=P, q_out=P, heads=0, freqs=P, positions=4, rotated=16) == 1
    assert append(c, s, q=P, q_out=P + 8, heads=4, freqs=P, positions=4, rotated=16) == 2


def test_attention_refuses():
    c, s = cache(), seqs()
    assert attend(c, s, q=None) == 1 and attend(c, s, o=None) == 1 and attend(c, s, strides=None) == 1
    assert attend(c, s, heads=3) == 1 and attend(c, s, heads=0) == 1
    assert attend(c, s, q=P + 4) == 2 and attend(c, s, strides=(256, 60) * 2) == 2 and attend(c, s, work=P + 8, size=1 << 20) == 2


def test_workspaces_follow_the_sizes():
    lib = _lib.load()
    need = lambda c, s, h: lib.mhip_paged_attention_workspace(C.byref(c), C.byref(s), h)  # noqa: E731
    assert need(cache(), seqs(), 3) == 0 and need(cache(), seqs(tokens=0), 4) == 0 and need(cache(heads=0), seqs(), 4) == 0
    assert 0 < need(cache(), seqs(), 4) < 64 << 20
    assert lib.mhip_token_log_probs_workspace(0, 50257, 20) == 0 and lib.mhip_token_log_probs_workspace(3, 500, 20) == 0
    assert 0 < lib.mhip_token_log_probs_workspace(3, 50257, 20) < 1 << 20


def test_log_probs_refuse():
    call = lambda x=P, t=P, p=P, e=P, tp=P, ti=P, rows=2, vocab=100, top=5, dt=BF16, tt=I32, w=None: _lib.load().mhip_token_log_probs(  # noqa: E731
        None, x, t, p, e, tp, ti, rows, vocab, top, dt, tt, w, 0)
    assert call(x=None) == 1 and call(t=None) == 1 and call(p=None) == 1 and call(tp=None) == 1 and call(ti=None) == 1
    assert call(rows=-1) == 1 and call(vocab=0) == 1 and call(top=65) == 1 and call(top=-1) == 1 and call(vocab=4) == 1
    assert call(dt=2) == 2 and call(tt=5) == 2 and call(x=P + 1) == 1 and call(w=P + 8) == 1
    assert call(rows=0, x=None) == 0


def test_host_tensors_are_refused():
    c = kernels.paged_cache(2, 2, 16, 64, torch.bfloat16, device="cpu")
    x, i = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: kernels.paged_append(c, x, x, i[None], i[:1], i), lambda: kernels.paged_attention(x, c, i[None], i[:1], i),
                 lambda: kernels.token_log_probs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="blocks of 16"):
        kernels.paged_cache(2, 2, 20, 64, torch.bfloat16, device="cpu")


def test_scale_bytes_of_the_oracle():
    for amax, byte in ((448.0, 127), (448.0001, 128), (1.0, 119), (1.75, 119), (1.7500001, 120), (0.0, 1), (1e-45, 1), (65504.0, 135)):
        assert scale_byte(amax) == byte
        assert amax <= 448 * 2.0 ** (byte - 127) and (byte == 1 or amax > 448 * 2.0 ** (byte - 128))
