"""Attention of sequences that have a prefix in common, against softmax over the prefix's keys and a sequence's own in float64."""
import ctypes

import numpy as np
import pytest
import torch

from tests.paged_util import HostCache, assert_within, half_step, table_of

gpu = pytest.mark.gpu
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
HALF = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def expected(q, cache, prefix, P, table, lengths, starts, scale=None, causal=True):
    """(result, bound) as paged_util.attention: what is left between the two launches is fp32, and joining adds 2^-22 at most."""
    u, (T, H, D), KV = half_step(q.dtype), q.shape, cache.x[0].shape[1]
    qd, scale = q.double().cpu().numpy(), D ** -0.5 if scale is None else scale
    out, bound = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    front = [cache.dense(w, np.asarray(prefix)[None], 0, P) for w in range(2)]
    for b, n in enumerate(lengths):
        k, v = (np.concatenate((front[w], cache.dense(w, table, b, n)), 1) for w in range(2))
        there = ~np.isnan(k[0]).any(1)
        m = starts[b + 1] - starts[b]
        rows = slice(starts[b], starts[b + 1])
        last = np.arange(n - m, n) if causal else np.full(m, n - 1)
        hidden = (np.arange(-P, n)[None] > np.where(np.arange(-P, n) < 0, P + n, last[:, None])) | ~there
        for h in range(H):
            kk, vv = np.nan_to_num(k[h // (H // KV)]), np.nan_to_num(v[h // (H // KV)])
            s = np.where(hidden, -np.inf, scale * (qd[rows, h] @ kk.T))
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(s - np.where(np.isinf(top), 0, top))
            p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
            out[rows, h] = p @ vv
            bound[rows, h] = 1.01 * (u * np.abs(out[rows, h]) + (u + 2.0 ** -13) * (p @ np.abs(vv))) + 1e-30
            if q.dtype == torch.float16:
                bound[rows, h] += 2.0 ** -25 * (2 + (P + n) * np.abs(vv).max(initial=0))
    return out, bound


def make(new, context, P, H, KV, D, page, dtype, eight, seed=0, width=None, pad=0, spread=1.0):
    rng = np.random.default_rng(seed)
    keys = [n + c for n, c in zip(new, context)]
    all_tables, pages = table_of(keys + [P], page, rng, max(width or 0, max(-(-n // page) for n in keys + [P]), 1))
    cache = HostCache(pages, KV, page, D, dtype, eight).fill(all_tables, keys + [P], rng, spread)
    table = all_tables[:-1, :width or max(1, max(-(-n // page) for n in keys))].copy()
    prefix = all_tables[-1, :max(-(-P // page), 1)].copy()
    starts = [0] + list(np.cumsum(new))
    q = torch.from_numpy(rng.standard_normal((starts[-1] + pad, H, D)).astype(np.float32)).to(dtype)
    return q, cache, prefix, table, keys, starts


def check(new, context, P, H, KV, D, page, dtype, eight, scale=None, causal=True, change=None, **kw):
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make(new, context, P, H, KV, D, page, dtype, eight, **kw)
    if change:
        change(prefix, table, cache)
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    args = (cache.to_device(), ints(prefix), ints([P]), ints(table), ints(keys), ints(starts))
    got = kernels.paged_attention_shared(q.cuda(), *args, scale=scale, is_causal=causal, out=out)
    assert got is out
    want, bound = expected(q, cache, prefix, P, table, keys, starts, scale, causal)
    assert_within(got[:starts[-1]], want[:starts[-1]], bound[:starts[-1]], f"{new} {context} {P}")
    assert (got[starts[-1]:] == 7).all()
    assert torch.equal(kernels.paged_attention_shared(q.cuda(), *args, scale=scale, is_causal=causal)[:starts[-1]], got[:starts[-1]])
    return got


@gpu
@HALF
@EIGHT
@pytest.mark.parametrize("H,KV,D,page", [(1, 1, 64, 16), (12, 12, 64, 16), (8, 2, 128, 64), (6, 2, 96, 32), (5, 1, 32, 128), (32, 2, 128, 256)], ids=str)
def test_a_token_a_sequence(H, KV, D, page, dtype, eight):
    for P in (1, 16, 77, 400):
        check([1] * 6, [0, 1, 15, 64, 200, 33], P, H, KV, D, page, dtype, eight, seed=P)


@gpu
@HALF
@EIGHT
@pytest.mark.parametrize("new", [[2, 1, 0, 5], [8, 3, 7, 4], [33, 1, 0, 70], [129, 128, 127, 1], [300, 270]], ids=str)
def test_several_tokens(new, dtype, eight):
    for causal, scale in ((True, None), (False, -0.07)):
        check(new, [0, 40, 30, 129][:len(new)], 333, 8, 4, 64, 16, dtype, eight, scale=scale, causal=causal, seed=len(new))
        check(new, [0, 40, 30, 129][:len(new)], 130, 4, 2, 128, 64, dtype, eight, scale=scale, causal=causal, seed=len(new))


@gpu
@EIGHT
@pytest.mark.parametrize("B", [1, 2, 7, 24, 33, 100])
def test_batches_of_any_size(B, eight):
    """One row to hundreds over the prefix, each kernel of it; more sequences than lanes."""
    check([1] * B, [(b * 37) % 90 for b in range(B)], 2500, 4, 1, 64, 32, torch.bfloat16, eight, seed=B)


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 5, 90])
def test_prefixes_of_no_keys_and_sequences_without_their_own(new, eight):
    """An empty prefix is none; a sequence may have nothing but the prefix, or nothing at all."""
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make([new] * 3, [20, 0, 300], 90, 4, 2, 64, 16, torch.bfloat16, eight)
    held = cache.to_device()
    none = kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([0]), ints(table), ints(keys), ints(starts))
    want, bound = expected(q, cache, prefix, 0, table, keys, starts)
    assert_within(none, want, bound)
    assert torch.equal(kernels.paged_attention_shared(q.cuda(), held, ints([]), ints([55]), ints(table), ints(keys), ints(starts)), none)
    short = [0, keys[1], 0]
    for P in (0, 90):
        got = kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([P]), ints(table), ints(short), ints(starts))
        want, bound = expected(q, cache, prefix, P, table, short, starts)
        assert_within(got, want, bound)
        if P == 0:
            assert (got[:new] == 0).all() and (got[2 * new:] == 0).all()
    lone = kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([90]), ints(np.zeros((3, 0))), ints(keys), ints(starts), is_causal=False)
    want, bound = expected(q, cache, prefix, 90, table, [0, 0, 0], [0] + list(np.cumsum([new] * 3)), causal=False)
    assert_within(lone, want, bound)


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 4, 100])
def test_padded_batches_and_absent_pages(new, eight):
    def holes(prefix, table, cache):
        prefix[2] = -1
        prefix[5] = 1 << 29
        table[0, 1] = -5
    check([new] * 3, [60, 20, 45], 120, 4, 2, 64, 16, torch.bfloat16, eight, pad=5, width=20, change=holes)


@gpu
def test_prefix_lengths_beyond_its_pages_and_starts_beyond_the_rows():
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make([3] * 3, [50, 20, 0], 96, 4, 2, 64, 16, torch.bfloat16, True)
    held = cache.to_device()
    want = kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([96]), ints(table), ints(keys), ints(starts))
    for P in (97, 1 << 30):
        assert torch.equal(kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([P]), ints(table), ints(keys), ints(starts)), want)
    kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([-9]), ints(table), ints(keys), ints(starts))
    assert torch.equal(kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([96]), ints(table), ints(keys), ints(starts[:3] + [1 << 20])), want)
    out = torch.full_like(q, 7, device="cuda")
    kernels.paged_attention_shared(q.cuda(), held, ints(prefix), ints([96]), ints(table), ints(keys), ints([0, 3, 3, 0]), out=out)
    assert torch.equal(out[:3], want[:3])


@gpu
@HALF
@pytest.mark.parametrize("new", [1, 40])
def test_large_scores(new, dtype):
    """Maxima of either part far above the other's."""
    for grow in ("prefix", "own"):
        def change(prefix, table, cache, grow=grow):
            for p in (prefix if grow == "prefix" else table.ravel()):
                if p >= 0:
                    cache.x[0][p] = (cache.x[0][p] * 6).to(dtype).float()        # (what the device's cache holds of them)
        check([new] * 3, [30, 90, 200], 150, 4, 2, 64, 16, dtype, False, change=change)


@gpu
@pytest.mark.parametrize("new", [1, 50])
def test_what_is_not_finite(new):
    """A NaN among the prefix's values reaches every row, in its element; one among a sequence's own the rows that see it."""
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make([new] * 3, [20, 60, 0], 90, 4, 2, 64, 16, torch.bfloat16, False)
    cache.x[1][table[1, 0], :, 3, 9] = float("inf")
    got = kernels.paged_attention_shared(q.cuda(), cache.to_device(), ints(prefix), ints([90]), ints(table), ints(keys), ints(starts))
    assert torch.isinf(got[starts[1]:starts[2], :, 9]).all() and torch.isfinite(got[:starts[1]]).all() and torch.isfinite(got[starts[2]:]).all()
    cache.x[1][prefix[3], :, 3, 5] = float("nan")
    got = kernels.paged_attention_shared(q.cuda(), cache.to_device(), ints(prefix), ints([90]), ints(table), ints(keys), ints(starts))
    assert torch.isnan(got[..., 5]).all() and torch.isfinite(torch.cat((got[..., :5], got[..., 6:9], got[..., 10:]), -1)).all()


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 3, 30, 140])
def test_views_in_place_and_workspaces(new, eight):
    """Queries in a projection, the result where they lie; the C entry with what suffices of the workspace, and with all of it."""
    from metalhlo_amd import _lib, kernels
    from tests.test_serving_host import Cache, Sequences
    lib = _lib.load()
    q, cache, prefix, table, keys, starts = make([new] * 3, [700, 60, 0], 900, 8, 2, 64, 16, torch.bfloat16, eight)
    held, T = cache.to_device(), q.shape[0]
    p, P, t, n, s = ints(prefix), ints([900]), ints(table), ints(keys), ints(starts)
    want, bound = expected(q, cache, prefix, 900, table, keys, starts)
    wide = torch.randn(T, 12 * 64, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 2 * 64:10 * 64].view(T, 8, 64)
    view.copy_(q)
    rest = wide[:, 10 * 64:].clone()
    assert kernels.paged_attention_shared(view, held, p, P, t, n, s, out=view) is view
    assert_within(view, want, bound)
    assert torch.equal(wide[:, 10 * 64:], rest)
    c = Cache(held.keys.data_ptr(), held.values.data_ptr(), *(0 if x is None else x.data_ptr() for x in held[2:]), *held.keys.shape)
    seqs = Sequences(t.data_ptr(), n.data_ptr(), s.data_ptr(), 3, t.shape[1], T)
    least = ctypes.c_int64()
    need = lib.mhip_paged_attention_shared_workspace(ctypes.byref(c), p.shape[0], ctypes.byref(seqs), 8, ctypes.byref(least))
    assert need > least.value > 0
    qd, room = q.cuda(), torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    strides = (ctypes.c_int64 * 4)(8 * 64, 64, 8 * 64, 64)
    for size in (least.value - 1, least.value, need - 1, need):
        out = torch.full_like(qd, 7)
        room.fill_(0xA5)
        rc = lib.mhip_paged_attention_shared(torch.cuda.current_stream().cuda_stream, ctypes.byref(c), p.data_ptr(), p.shape[0], P.data_ptr(), ctypes.byref(seqs), qd.data_ptr(), out.data_ptr(), 8, 0.125, 1,
                                             strides, kernels.DTYPE_CODE[torch.bfloat16], room.data_ptr(), size)
        assert rc == (1 if size < least.value else 0)
        if rc == 0:
            assert_within(out, want, bound, str(size))
            assert (room[size:] == 0xA5).all()


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 30])
def test_other_streams_and_graphs(new, eight):
    """A captured call serves the prefix and the lengths that are there when it is replayed."""
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make([new] * 4, [300, 60, 0, 90], 500, 8, 2, 64, 16, torch.bfloat16, eight)
    held, qd = cache.to_device(), q.cuda()
    p, P, t, n, s = ints(prefix), ints([500]), ints(table), ints(keys), ints(starts)
    want = kernels.paged_attention_shared(qd, held, p, P, t, n, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = kernels.paged_attention_shared(qd, held, p, P, t, n, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.paged_attention_shared(qd, held, p, P, t, n, s)
        again = kernels.paged_attention_shared(qd, held, p, P, t, n, s, is_causal=False)
    for turn in range(3):
        P.fill_(500 - 160 * turn)
        n[0] = keys[0] - 100 * turn
        qd.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)).to(q.dtype))
        graph.replay()
        assert torch.equal(got, kernels.paged_attention_shared(qd, held, p, P, t, n, s)) and torch.equal(again, kernels.paged_attention_shared(qd, held, p, P, t, n, s, is_causal=False))


@gpu
def test_refusals():
    from metalhlo_amd import kernels
    q, cache, prefix, table, keys, starts = make([2] * 3, [30, 6, 0], 90, 4, 2, 64, 16, torch.bfloat16, True)
    held, qd = cache.to_device(), q.cuda()
    p, P, t, n, s = ints(prefix), ints([90]), ints(table), ints(keys), ints(starts)
    assert kernels.paged_attention_shared(qd[:0], held, p, P, t, n, s).shape == (0, 4, 64)
    for args, error in [((qd, held, p.long(), P, t, n, s), TypeError), ((qd, held, p[None], P, t, n, s), ValueError), ((qd, held, p, ints([1, 2]), t, n, s), ValueError), ((qd, held, p, P.float(), t, n, s), TypeError),
                        ((qd, held, p.cpu(), P, t, n, s), RuntimeError), ((qd[:, :3], held, p, P, t, n, s), ValueError), ((qd.float(), held, p, P, t, n, s), TypeError), ((qd, held, p, P, t, n[:2], s), ValueError),
                        ((qd, held, p[::2], P, t, n, s), ValueError)]:
        with pytest.raises(error):
            kernels.paged_attention_shared(*args)
    with pytest.raises(ValueError):
        kernels.paged_attention_shared(qd, held, p, P, t, n, s, out=qd[:1])


def test_refusals_of_the_entry_point(lib):
    from tests.test_serving_host import Cache, Sequences
    base_c, base_s = dict(keys=16, values=16, ks=None, vs=None, pages=4, heads=2, page=16, D=32), dict(table=16, lengths=16, starts=16, B=2, width=3, T=5)

    def go(prefix=16, width=3, P=16, q=16, o=16, H=4, strides=True, dtype=3, work=16, size=1 << 30, c={}, s={}):
        st = (ctypes.c_int64 * 4)(128, 32, 128, 32) if strides is True else strides
        return lib.mhip_paged_attention_shared(None, ctypes.byref(Cache(*{**base_c, **c}.values())), prefix, width, P, ctypes.byref(Sequences(*{**base_s, **s}.values())), q, o, H, 1.0, 1, st, dtype, work, size)

    assert go(prefix=None) == 1 and go(P=None) == 1 and go(width=-1) == 1 and go(q=None) == 1 and go(H=3) == 1 and go(strides=None) == 1 and go(work=None) == 1 and go(size=64) == 1
    assert go(width=1 << 21) == 2 and go(dtype=1) == 2 and go(work=8) == 2 and go(strides=(ctypes.c_int64 * 4)(4, 32, 128, 32)) == 2 and go(c=dict(page=24)) == 2
    assert go(s=dict(T=0)) == 0 and go(s=dict(B=0)) == 0
