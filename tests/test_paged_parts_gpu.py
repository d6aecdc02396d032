"""The operators on a paged cache where a launch's work is dealt over workgroups: parts of tiles of every form, whole tiles without a workspace, many sequences, starts that are
none, calls side by side; and what the compiler made of their kernels."""
import ctypes
import os

import numpy as np
import pytest
import torch

from tests.paged_util import HostCache, assert_within, attention, attention_at_once, table_of
from tests.util import NAME

gpu = pytest.mark.gpu
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def _batch(new, context, H, KV, D, page, dtype, eight, seed=0, width=None):
    rng = np.random.default_rng(seed)
    keys = [n + c for n, c in zip(new, context)]
    table, pages = table_of(keys, page, rng, width)
    cache = HostCache(pages, KV, page, D, dtype, eight).fill(table, keys, rng)
    starts = [0] + list(np.cumsum(new))
    q = torch.from_numpy(rng.standard_normal((starts[-1], H, D)).astype(np.float32)).to(dtype)
    return q, cache, table, keys, starts


def _call(q, held, table, keys, starts, scale, causal, out, workspace=None):
    """The C entry point itself, with a workspace or none."""
    from metalhlo_amd import _lib, kernels
    from tests.test_serving_host import Cache, Sequences
    lib = _lib.load()
    T, H, D = q.shape
    c = Cache(held.keys.data_ptr(), held.values.data_ptr(), *(0 if s is None else s.data_ptr() for s in held[2:]), held.keys.shape[0], held.keys.shape[1], held.keys.shape[2], D)
    s = Sequences(table.data_ptr(), keys.data_ptr(), starts.data_ptr(), keys.shape[0], table.shape[1], T)
    strides = (ctypes.c_int64 * 4)(q.stride(0), q.stride(1), out.stride(0), out.stride(1))
    need = lib.mhip_paged_attention_workspace(ctypes.byref(c), ctypes.byref(s), H)
    _lib.check(lib.mhip_paged_attention(torch.cuda.current_stream().cuda_stream, ctypes.byref(c), ctypes.byref(s), q.data_ptr(), out.data_ptr(), H, scale, int(causal), strides,
                                        kernels.DTYPE_CODE[q.dtype], 0 if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel()))
    return need


# rows of a sequence on average: up to 16 and up to 32, one token and several, 128 and 256
FORMS = [("one token", [1] * 5, 4, 2, 64, 16), ("one token, many heads", [1] * 4, 20, 1, 96, 32), ("several", [4, 2, 6, 3], 4, 2, 128, 64), ("twenty", [20, 25, 3, 30], 1, 1, 32, 16),
         ("tiles", [150, 1, 90, 257], 2, 1, 64, 16), ("large tiles", [300, 420, 1, 280], 2, 1, 128, 64)]
form = pytest.mark.parametrize("what,new,H,KV,D,page", FORMS, ids=[f[0] for f in FORMS])


@gpu
@EIGHT
@form
def test_dealt_over_parts(what, new, H, KV, D, page, eight):
    """Contexts of thousands of keys next to none; the same twice."""
    from metalhlo_amd import kernels
    context = [2900, 0, 5003, 1700, 61][:len(new)]
    q, cache, table, keys, starts = _batch(new, context, H, KV, D, page, torch.bfloat16, eight, seed=D)
    held, args = cache.to_device(), (ints(table), ints(keys), ints(starts))
    for causal, scale in ((True, None), (False, -0.07)):
        got = kernels.paged_attention(q.cuda(), held, *args, scale=scale, is_causal=causal)
        want, bound = attention_at_once(q, cache, table, keys, starts, scale, causal)
        assert_within(got, want, bound, f"{what} {causal}")
        assert torch.equal(kernels.paged_attention(q.cuda(), held, *args, scale=scale, is_causal=causal), got)


@gpu
@EIGHT
@form
def test_without_a_workspace(what, new, H, KV, D, page, eight):
    context = [1400, 0, 300, 1700, 61][:len(new)]
    q, cache, table, keys, starts = _batch(new, context, H, KV, D, page, torch.float16, eight, seed=D + 1)
    held, qd = cache.to_device(), q.cuda()
    out = torch.full_like(qd, 7)
    need = _call(qd, held, ints(table), ints(keys), ints(starts), D ** -0.5, True, out)
    assert need > 0
    want, bound = attention_at_once(q, cache, table, keys, starts)
    assert_within(out, want, bound, what)
    # one that is a byte too small is none; one that is large enough holds anything beforehand, and words behind its end stay
    room = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    other = torch.full_like(qd, 7)
    _call(qd, held, ints(table), ints(keys), ints(starts), D ** -0.5, True, other, room[:need - 1])
    assert torch.equal(other, out) and (room == 0xA5).all()
    _call(qd, held, ints(table), ints(keys), ints(starts), D ** -0.5, True, other, room[:need])
    assert_within(other, want, bound, what)
    assert (room[need:] == 0xA5).all()


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 3, 40])
def test_more_sequences_than_lanes(new, eight):
    """Sequences behind the 64th, empty ones among them, and those without tokens."""
    from metalhlo_amd import kernels
    B = 150
    news = [new if b % 7 else 0 for b in range(B)]
    context = [1 + (b * 37) % 400 + (3000 if b in (70, 149) else 0) for b in range(B)]
    q, cache, table, keys, starts = _batch(news, context, 4, 2, 32, 16, torch.bfloat16, eight, seed=new)
    got = kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts))
    want, bound = attention_at_once(q, cache, table, keys, starts)
    assert_within(got, want, bound)


@gpu
@EIGHT
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
def test_parts_with_holes_and_wild_values(D, page, eight):
    """Parts of tiles whose pages the table does not name, and a NaN among the values of a new token: rows in front of it are finite, the others NaN in that element alone."""
    from metalhlo_amd import kernels
    new, context = [300, 330], [3000, 2500]
    q, cache, table, keys, starts = _batch(new, context, 2, 1, D, page, torch.bfloat16, eight, seed=9)
    for b in range(2):
        table[b, [3, 17, (2000 + 300 * b) // page]] = -1
    rows = [0, 1, 150, 299, 300, 301, 500, 629]
    wild = [3200, 2700]
    for b in range(2):
        cache.x[1][table[b, wild[b] // page], :, wild[b] % page, 5] = float("nan")
    got = kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts)).double().cpu().numpy()
    seen = np.array([r - starts[b] + context[b] >= wild[b] for b in range(2) for r in range(starts[b], starts[b + 1])])
    assert np.isnan(got[seen][:, :, 5]).all() and np.isfinite(np.delete(got, 5, 2)).all() and np.isfinite(got[~seen]).all()
    # the oracle for a few rows: the sequence cut behind each row's token
    for b in range(2):
        cache.x[1][table[b, wild[b] // page], :, wild[b] % page, 5] = 0.0
    for r in rows:
        b = int(r >= starts[1])
        n = context[b] + r - starts[b] + 1
        want, bound = attention(q[r:r + 1], cache, table[b:b + 1], [n], [0, 1])
        ok = np.ones(D, bool)
        ok[5] = not seen[r]
        assert (np.abs(got[r:r + 1] - want) <= bound)[:, :, ok].all(), r


@gpu
@EIGHT
def test_scales_of_any_sign(eight):
    from metalhlo_amd import kernels
    for new, context in (([1, 1], [300, 40]), ([70, 30], [300, 0])):
        q, cache, table, keys, starts = _batch(new, context, 4, 2, 64, 16, torch.bfloat16, eight)
        for scale in (-0.125, 0.0, 2.0 ** -30):
            got = kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts), scale=scale)
            want, bound = attention_at_once(q, cache, table, keys, starts, scale)
            assert_within(got, want, bound, str(scale))


@gpu
@pytest.mark.parametrize("new", [1, 4, 100])
def test_starts_beyond_the_rows(new):
    """Starts below zero, behind the call's rows or falling are held to them: sequences that have their rows are answered, and nothing else is written."""
    from metalhlo_amd import kernels
    q, cache, table, keys, starts = _batch([new] * 3, [50, 20, 2000], 4, 2, 64, 16, torch.bfloat16, True)
    held, T = cache.to_device(), starts[-1]
    want, bound = attention_at_once(q, cache, table, keys, starts)
    for bad in ([-9, new, 2 * new, T + 1000], [0, new, 2 * new, 2 ** 31 - 1]):
        got = kernels.paged_attention(q.cuda(), held, ints(table), ints(keys), ints(bad))
        assert_within(got, want, bound)
    out = torch.full((T, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kernels.paged_attention(q.cuda(), held, ints(table), ints(keys), ints([0, new, new - 1, new - 1]), out=out)
    assert_within(out[:new], want[:new], bound[:new])
    assert (out[new:] == 7).all()


@gpu
def test_calls_side_by_side():
    """Two streams at once, each with its own batch; every call is right however they meet."""
    from metalhlo_amd import kernels
    jobs = []
    for seed, (new, context, H, KV, D, page) in enumerate((([1] * 6, [4000, 10, 3000, 900, 0, 5000], 8, 2, 64, 16), ([200, 90], [3000, 2500], 4, 2, 64, 64))):
        q, cache, table, keys, starts = _batch(new, context, H, KV, D, page, torch.bfloat16, bool(seed), seed=seed)
        args = (q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts))
        jobs.append((torch.cuda.Stream(), args, kernels.paged_attention(*args)))
    x = torch.randn(3, 50257, device="cuda").bfloat16()
    tokens = ints([5, 50256, 0])
    scored = kernels.token_log_probs(x, tokens, top=20)
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(20):
        for i, (stream, args, _) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[i].append((kernels.paged_attention(*args), kernels.token_log_probs(x, tokens, top=20)))
    torch.cuda.synchronize()
    for i, (_, _, want) in enumerate(jobs):
        assert all(torch.equal(a, want) and all(torch.equal(s, t) for s, t in zip(b, scored)) for a, b in got[i])


@gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(3, 50257, torch.bfloat16), (1, 20001, torch.float32), (64, 9000, torch.float16)], ids=lambda v: str(NAME.get(v, v)))
def test_log_probs_without_a_workspace(rows, vocab, dtype):
    """A row that no workspace is there for is one workgroup's; sums in another order, alternatives the same."""
    from metalhlo_amd import _lib, kernels
    lib = _lib.load()
    x = torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dtype)
    tokens = ints([7] * rows)
    want = kernels.token_log_probs(x, tokens, top=9)
    assert lib.mhip_token_log_probs_workspace(rows, vocab, 9) > 0
    got = [torch.full_like(t, 5) for t in want]
    _lib.check(lib.mhip_token_log_probs(torch.cuda.current_stream().cuda_stream, x.data_ptr(), tokens.data_ptr(), *(t.data_ptr() for t in got), rows, vocab, 9, kernels.DTYPE_CODE[dtype],
                                        kernels.DTYPE_CODE[torch.int32], 0, 0))
    assert torch.equal(got[3], want[3])
    # log l of sums of vocab / 256 weights a lane and of less: 2^-24 of the sum for each
    for a, b in zip(got[:3], want[:3]):
        assert ((a - b).abs() <= 2.0 ** -24 * (vocab / 128 + 64) * (2 + b.abs())).all()


@gpu
@EIGHT
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 2, 4], [200, 1, 150]], ids=str)
def test_pages_far_into_a_cache(new, eight):
    """Bytes beyond 2^32 of a cache, and rows of queries as far apart: the same bits as in a small cache."""
    try:
        _far(new, eight)
    finally:
        torch.cuda.empty_cache()                # (gigabytes, which a later test's small tensor would keep from going back)


def _far(new, eight):
    from metalhlo_amd import kernels
    KV, page, D, pages = 8, 64, 128, 70000
    keys = [n + c for n, c in zip(new, (100, 3, 1500))]
    T, starts = sum(new), ints([0] + list(np.cumsum(new)))
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(T, KV, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    far_q = torch.empty_strided((T, 2 * KV, D), (2 ** 31 // T // 64 * 64 + 64, D, 1), dtype=torch.bfloat16, device="cuda")
    q = torch.randn(T, 2 * KV, D, device="cuda", generator=g).bfloat16()
    far_q.copy_(q)
    freqs = torch.randn(2000, D, device="cuda", generator=g)
    count = [-(-n // page) for n in keys]
    table = -np.ones((3, max(count)), dtype=np.int32)
    for b, c in enumerate(count):
        table[b, :c] = sum(count[:b]) + np.arange(c)
    results = []
    for size, first in ((sum(count), 0), (pages, pages - sum(count))):
        cache = kernels.paged_cache(size, KV, page, D, torch.float8_e4m3fn if eight else torch.bfloat16)
        held = [t[first:] for t in cache if t is not None]
        for t in held:
            t.view(torch.uint8).fill_(40)
        t = ints(np.where(table < 0, table, table + first))
        turned = kernels.paged_append(cache, k, v, t, ints(keys), starts, q=far_q if first else q, freqs=freqs, out=far_q if first else None)
        o = kernels.paged_attention(turned, cache, t, ints(keys), starts)
        results.append([turned.contiguous(), o] + [h.view(torch.uint8).clone() for h in held])
        del cache, held
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[0][1].isfinite().all())


@gpu
@pytest.mark.parametrize("T", [3, 40, 300])
def test_a_table_without_columns(T):
    """No sequence can have keys: zeros, and nothing is stored."""
    from metalhlo_amd import kernels
    cache = kernels.paged_cache(4, 2, 16, 64, torch.bfloat16)
    cache.keys.fill_(3)
    q, k = torch.ones(T, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(T, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    args = (table, ints([5, 0, T]), ints([0, 1, 1, T]))
    kernels.paged_append(cache, k, k, *args)
    assert (cache.keys == 3).all()
    for causal in (True, False):
        assert (kernels.paged_attention(q, cache, *args, is_causal=causal) == 0).all()


@gpu
@pytest.mark.parametrize("rows,vocab,dtype,top", [(300, 32003, torch.float32, 5), (400, 9001, torch.bfloat16, 64), (512, 4096, torch.float16, 1), (7, 300001, torch.float32, 20)],
                         ids=lambda v: str(NAME.get(v, v)))
def test_log_probs_of_some_hundred_rows(rows, vocab, dtype, top):
    from tests.test_token_log_probs_gpu import _check, _logits
    _check(*_logits(rows, vocab, dtype, rows), top, str((rows, vocab, top)))


@pytest.mark.parametrize("name", ["paged_rows_kernel", "paged_tile_kernel", "paged_append_kernel", "append_few_kernel", "token_log_probs_kernel"])
def test_nothing_is_kept_in_scratch(name):
    """Scratch memory costs a launch of these 10 us, whatever its size."""
    pytest.importorskip("msgpack")
    from tests.test_kernel_resources import LIB, _kernels
    if not os.path.exists(LIB):
        pytest.skip("no built library")
    found = [k for k in _kernels() if name in k[".name"]]
    assert found
    assert [k[".name"] for k in found if k[".private_segment_fixed_size"] or k[".vgpr_spill_count"]] == []
