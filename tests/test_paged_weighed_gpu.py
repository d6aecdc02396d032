"""Attention that adds up the weights it gives, against softmax in float64; a sequence of decode steps with evictions in between.

Bounds.  A weight is off by what its score and its row's sum are off by: 2^-13 each (paged_util.attention), so 2^-12 of itself; adding R of them and what was there in fp32 costs (R + 2) 2^-24 of the sum at most."""
import ctypes

import numpy as np
import pytest
import torch

from tests.paged_util import HostCache, assert_within, attention_at_once, table_of

gpu = pytest.mark.gpu
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
HALF = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def given(q, cache, table, lengths, starts, scale=None, causal=True):
    """[heads, keys] of each sequence: the weights that its tokens give."""
    (T, H, D), KV = q.shape, cache.x[0].shape[1]
    qd, scale, out = q.double().cpu().numpy(), D ** -0.5 if scale is None else scale, []
    for b, n in enumerate(lengths):
        k, m = cache.dense(0, table, b, n), starts[b + 1] - starts[b]
        there = ~np.isnan(k[0]).any(1)
        hidden = (np.arange(n)[None] > (np.arange(n - m, n) if causal else np.full(m, n))[:, None]) | ~there
        total = np.zeros((KV, n))
        for h in range(H):
            s = np.where(hidden, -np.inf, scale * (qd[starts[b]:starts[b + 1], h] @ np.nan_to_num(k[h // (H // KV)]).T))
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(s - np.where(np.isinf(top), 0, top))
            total[h // (H // KV)] += (p / np.maximum(p.sum(1, keepdims=True), 1e-300)).sum(0)
        out.append(total)
    return out


def make(new, context, H, KV, D, page, dtype, eight, seed=0, width=None, pad=0, spread=1.0):
    rng = np.random.default_rng(seed)
    keys = [n + c for n, c in zip(new, context)]
    table, pages = table_of(keys, page, rng, width)
    cache = HostCache(pages, KV, page, D, dtype, eight).fill(table, keys, rng, spread)
    starts = [0] + list(np.cumsum(new))
    q = torch.from_numpy(rng.standard_normal((starts[-1] + pad, H, D)).astype(np.float32)).to(dtype)
    weights = torch.from_numpy(rng.random((pages, KV, page), np.float32) * 3)
    return q, cache, table, keys, starts, weights


def expected_weights(before, q, cache, table, keys, starts, scale=None, causal=True):
    """(weights, bound) [pages, heads, page] in float64; slots that nothing is added to are as they were, to the bit."""
    page, want, bound = before.shape[2], before.double().numpy().copy(), np.zeros(before.shape)
    G = q.shape[1] // before.shape[1]
    for b, total in enumerate(given(q, cache, table, keys, starts, scale, causal)):
        m = starts[b + 1] - starts[b]
        if m == 0:
            continue
        for i in range(keys[b]):
            p = int(table[b, i // page]) if i // page < table.shape[1] else -1
            if not 0 <= p < before.shape[0]:
                continue
            old = want[p, :, i % page] if i < keys[b] - m else 0.0
            want[p, :, i % page] = old + total[:, i]
            bound[p, :, i % page] = 2.0 ** -12 * total[:, i] + (m * G + 2) * 2.0 ** -24 * (old + total[:, i]) + 1e-30
    return want, bound


def check(new, context, H, KV, D, page, dtype, eight, scale=None, causal=True, change=None, **kw):
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make(new, context, H, KV, D, page, dtype, eight, **kw)
    if change:
        change(table, cache)
    held, weights, qd = cache.to_device(), before.cuda(), q.cuda()
    args = (ints(table), ints(keys), ints(starts))
    got = kernels.paged_attention_weighed(qd, held, weights, *args, scale=scale, is_causal=causal)
    n = starts[-1]
    assert torch.equal(got[:n], kernels.paged_attention(qd, held, *args, scale=scale, is_causal=causal)[:n])
    want, bound = expected_weights(before, q, cache, table, keys, starts, scale, causal)
    off = np.abs(weights.double().cpu().numpy() - want)
    assert (off <= bound).all(), (off - bound).max()
    again = before.cuda()
    kernels.paged_attention_weighed(qd, held, again, *args, scale=scale, is_causal=causal)
    assert torch.equal(again, weights)


@gpu
@HALF
@EIGHT
@pytest.mark.parametrize("H,KV,D,page", [(1, 1, 64, 16), (12, 12, 64, 16), (8, 2, 128, 64), (6, 2, 96, 32), (5, 1, 32, 128), (32, 2, 128, 256)], ids=str)
def test_one_token(H, KV, D, page, dtype, eight):
    check([1] * 9, [0, 14, 15, 16, 62, 63, 64, 199, 1030], H, KV, D, page, dtype, eight, seed=D + page)


@gpu
@HALF
@EIGHT
@pytest.mark.parametrize("new", [[2, 1, 0, 5], [8, 3, 7, 4], [33, 1, 0, 70], [129, 128, 127, 1], [300, 270]], ids=str)
def test_several_tokens(new, dtype, eight):
    for causal, scale in ((True, None), (False, -0.07)):
        check(new, [0, 40, 30, 129][:len(new)], 8, 4, 64, 16, dtype, eight, scale=scale, causal=causal, seed=len(new))
        check(new, [0, 40, 30, 129][:len(new)], 4, 2, 128, 64, dtype, eight, scale=scale, causal=causal, seed=len(new))


@gpu
@EIGHT
@pytest.mark.parametrize("D,page", [(32, 32), (96, 64), (128, 128), (128, 16)], ids=str)
def test_whole_prompts(D, page, eight):
    check([400, 17, 256], [0, 0, 0], 6, 2, D, page, torch.bfloat16, eight, seed=D)


@gpu
@EIGHT
@pytest.mark.parametrize("new,H", [(1, 4), (1, 20), (5, 4), (40, 2)])
def test_long_caches_and_many_sequences(new, H, eight):
    check([new] * 4, [5003, 0, 2900, 61], H, 1, 64, 32, torch.bfloat16, eight)
    check([new if b % 7 else 0 for b in range(90)], [(b * 37) % 300 for b in range(90)], H, 1, 32, 16, torch.bfloat16, eight)


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 4, 100])
def test_padded_batches_absent_pages_and_wide_tables(new, eight):
    def holes(table, cache):
        table[0, 1], table[2, 0], table[1, 2] = -5, 1 << 29, -1
    check([new] * 3, [60, 20, 45], 4, 2, 64, 16, torch.bfloat16, eight, pad=5, width=20, change=holes)


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 3, 90])
def test_slots_that_hold_no_key_stay(new, eight):
    """What lies behind a sequence's last key, and weights of pages that belong to none, keep their bits, a NaN among them; so do those of the call's own tokens not, which begin at zero."""
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([new] * 2, [37, 70], 4, 2, 64, 32, torch.bfloat16, eight)
    spare = [p for p in range(before.shape[0]) if p not in set(table.ravel())]
    before[spare] = float("nan")
    for b in range(2):
        before[table[b, (keys[b] - 1) // 32], :, (keys[b] - 1) % 32 + 1:] = float("nan")
        for i in range(keys[b] - new, keys[b]):
            before[table[b, i // 32], :, i % 32] = float("nan")
    weights = before.cuda()
    kernels.paged_attention_weighed(q.cuda(), cache.to_device(), weights, ints(table), ints(keys), ints(starts))
    now, held = weights.cpu(), torch.zeros(before.shape, dtype=torch.bool)
    for b in range(2):
        for i in range(keys[b]):
            held[table[b, i // 32], :, i % 32] = True
    assert torch.isfinite(now[held]).all() and torch.equal(now[~held].view(torch.int32), before[~held].view(torch.int32))


@gpu
@HALF
@pytest.mark.parametrize("new", [1, 40])
def test_large_scores(new, dtype):
    """Rows whose weight is one key's: the sums of weights are the number of rows."""
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([new] * 3, [30, 90, 200], 4, 2, 64, 16, dtype, False, spread=20.0)
    weights = torch.zeros_like(before).cuda()
    kernels.paged_attention_weighed(q.cuda(), cache.to_device(), weights, ints(table), ints(keys), ints(starts))
    for b in range(3):
        total = sum(weights[int(table[b, i // 16]), :, i % 16].double() for i in range(keys[b])).cpu()
        assert ((total - 2 * new).abs() <= 2 * new * 2.0 ** -12).all()


@gpu
@pytest.mark.parametrize("new", [1, 50])
def test_a_nan_stays_with_its_row(new):
    """A query that is not finite gives the keys that it sees NaN, and those of other heads and sequences none."""
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([new] * 3, [30, 90, 20], 4, 2, 64, 16, torch.bfloat16, True)
    q[starts[1], 1, 5] = float("nan")
    weights = before.cuda()
    kernels.paged_attention_weighed(q.cuda(), cache.to_device(), weights, ints(table), ints(keys), ints(starts))
    w = weights.cpu()
    for b in range(3):
        for i in range(keys[b]):
            at = w[int(table[b, i // 16]), :, i % 16]
            assert bool(torch.isnan(at[0])) == (b == 1 and i <= 90) and torch.isfinite(at[1])


@gpu
@pytest.mark.parametrize("new", [1, 3, 130])
def test_starts_and_lengths_beyond(new):
    """Starts behind the call's rows and lengths beyond the table are held to them."""
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([new] * 3, [50, 20, 100], 4, 2, 64, 16, torch.bfloat16, True)
    held, qd = cache.to_device(), q.cuda()
    one, two = before.cuda(), before.cuda()
    kernels.paged_attention_weighed(qd, held, one, ints(table), ints(keys), ints(starts))
    kernels.paged_attention_weighed(qd, held, two, ints(table), ints(keys), ints(starts[:3] + [1 << 20]))
    assert torch.equal(one, two)
    far = keys[:2] + [table.shape[1] * 16 + 7]
    three = before.cuda()
    got = kernels.paged_attention_weighed(qd, held, three, ints(table), ints(far), ints(starts))
    same = kernels.paged_attention(qd, held, ints(table), ints(far), ints(starts))       # (NaN where the length reaches slots that no token has been to)
    assert torch.equal(torch.isnan(got), torch.isnan(same)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(same))
    kernels.paged_attention_weighed(qd, held, three, ints(table), ints([-3, 1 << 30, 0]), ints([5, -1, 1 << 30, 2]))
    none = before.cuda()
    kernels.paged_attention_weighed(qd, held, none, ints(np.zeros((3, 0))), ints(keys), ints(starts))
    assert torch.equal(none.cpu(), before)


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 3, 30, 140])
def test_views_and_workspaces(new, eight):
    from metalhlo_amd import _lib, kernels
    from tests.test_serving_host import Cache, Sequences
    lib = _lib.load()
    q, cache, table, keys, starts, before = make([new] * 3, [1700, 60, 0], 8, 2, 64, 16, torch.bfloat16, eight)
    held, T = cache.to_device(), q.shape[0]
    t, n, s = ints(table), ints(keys), ints(starts)
    wide = torch.randn(T, 12 * 64, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 2 * 64:10 * 64].view(T, 8, 64)
    view.copy_(q)
    weights = before.cuda()
    whole = kernels.paged_attention_weighed(view, held, weights, t, n, s)
    want, bound = expected_weights(before, q, cache, table, keys, starts)
    assert (np.abs(weights.double().cpu().numpy() - want) <= bound).all()
    rows, limit = attention_at_once(q, cache, table, keys, starts)
    assert_within(whole, rows, limit)
    c = Cache(held.keys.data_ptr(), held.values.data_ptr(), *(0 if x is None else x.data_ptr() for x in held[2:]), *held.keys.shape)
    seqs = Sequences(t.data_ptr(), n.data_ptr(), s.data_ptr(), 3, t.shape[1], T)
    least = ctypes.c_int64()
    need = lib.mhip_paged_attention_weighed_workspace(ctypes.byref(c), ctypes.byref(seqs), 8, ctypes.byref(least))
    assert need > least.value > 0
    qd, room = q.cuda(), torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    strides = (ctypes.c_int64 * 4)(8 * 64, 64, 8 * 64, 64)
    for size in (least.value - 1, least.value, need - 1, need):
        out, weights = torch.full_like(qd, 7), before.cuda()
        room.fill_(0xA5)
        rc = lib.mhip_paged_attention_weighed(torch.cuda.current_stream().cuda_stream, ctypes.byref(c), ctypes.byref(seqs), qd.data_ptr(), out.data_ptr(), weights.data_ptr(), 8, 0.125, 1, strides,
                                              kernels.DTYPE_CODE[torch.bfloat16], room.data_ptr(), size)
        assert rc == (1 if size < least.value else 0)
        if rc == 0:
            assert_within(out, rows, limit, str(size))
            assert (np.abs(weights.double().cpu().numpy() - want) <= bound).all() and (room[size:] == 0xA5).all()


@gpu
@EIGHT
@pytest.mark.parametrize("new", [1, 30])
def test_other_streams_and_graphs(new, eight):
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([new] * 4, [300, 60, 0, 90], 8, 2, 64, 16, torch.bfloat16, eight)
    held, qd, weights = cache.to_device(), q.cuda(), before.cuda()
    t, n, s = ints(table), ints(keys), ints(starts)
    want = kernels.paged_attention_weighed(qd, held, weights, t, n, s)
    other, side = before.cuda(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = kernels.paged_attention_weighed(qd, held, other, t, n, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want) and torch.equal(other, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.paged_attention_weighed(qd, held, weights, t, n, s)
    for turn in range(3):
        n[0] = keys[0] - 100 * turn
        qd.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)).to(q.dtype))
        weights.copy_(before)
        graph.replay()
        other.copy_(before)
        assert torch.equal(got, kernels.paged_attention_weighed(qd, held, other, t, n, s)) and torch.equal(weights, other)


@gpu
@EIGHT
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,row", [(2, 0), (3, 0), (3, 1), (4, 2), (9, 3), (9, 5)])
def test_a_row_that_is_not_finite_gives_later_keys_nothing(new, row, what, eight):
    """Of a prompt's tokens one whose scores are not finite: the keys that it sees get NaN, those of later tokens do not, whether the scores are kept in the workspace or formed again."""
    from metalhlo_amd import _lib, kernels
    from tests.test_serving_host import Cache, Sequences
    lib = _lib.load()
    for context in (28, 29, 30, 31):
        q, cache, table, keys, starts, before = make([new] * 2, [20, context], 4, 2, 64, 16, torch.bfloat16, eight, width=8)
        q[starts[1] + row, 1, 5] = what
        held, qd, t, n, s = cache.to_device(), q.cuda(), ints(table), ints(keys), ints(starts)
        c = Cache(held.keys.data_ptr(), held.values.data_ptr(), *(0 if x is None else x.data_ptr() for x in held[2:]), *held.keys.shape)
        seqs = Sequences(t.data_ptr(), n.data_ptr(), s.data_ptr(), 2, 8, 2 * new)
        least = ctypes.c_int64()
        need = lib.mhip_paged_attention_weighed_workspace(ctypes.byref(c), ctypes.byref(seqs), 4, ctypes.byref(least))
        assert need > least.value > 0
        room, strides = torch.empty(need, dtype=torch.uint8, device="cuda"), (ctypes.c_int64 * 4)(4 * 64, 64, 4 * 64, 64)
        for size in (least.value, need):
            out, weights = torch.empty_like(qd), before.cuda()
            _lib.check(lib.mhip_paged_attention_weighed(torch.cuda.current_stream().cuda_stream, ctypes.byref(c), ctypes.byref(seqs), qd.data_ptr(), out.data_ptr(), weights.data_ptr(), 4, 0.125, 1,
                                                        strides, kernels.DTYPE_CODE[torch.bfloat16], room.data_ptr(), size))
            w = weights.cpu()
            for b in range(2):
                for i in range(keys[b]):
                    at = w[int(table[b, i // 16]), :, i % 16]
                    assert bool(torch.isnan(at[0])) == (b == 1 and i <= context + row) and torch.isfinite(at[1]), (context, size == need, b, i)


@gpu
@pytest.mark.parametrize("dtype,eight", [(torch.bfloat16, False), (torch.float16, True)], ids=["bf16", "f16 8bit"])
def test_a_run_of_steps(dtype, eight):
    """Prompts, decode steps and evictions as a program takes them, behind a prefix in common and with 4-bit projections: every step's operators against plain ones over the keys that are left."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(5)
    H, KV, D, page, B, M = 4, 2, 64, 16, 3, 96
    normal = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype).cuda()  # noqa: E731
    w_qkv = kernels.quantize_w4(normal(M, (H + 2 * KV) * D) * 0.1, 32, dtype)
    w_out = kernels.quantize_w4(normal(H * D, M) * 0.1, 64, dtype)
    cache = kernels.paged_cache(80, KV, page, D, torch.float8_e4m3fn if eight else dtype)
    weights = torch.full((80, KV, page), float("nan"), device="cuda")
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(B, 20)
    prefix, P = torch.arange(60, 70, dtype=torch.int32, device="cuda"), ints([150])
    kernels.paged_append(cache, normal(150, KV, D), normal(150, KV, D), prefix[None], P, ints([0, 150]))
    lengths = [0] * B
    for step, new in enumerate(([70, 33, 120], [1, 1, 1], [1, 1, 1], [9, 1, 4], [1, 1, 1])):
        T = sum(new)
        lengths = [n + m for n, m in zip(lengths, new)]
        starts = ints([0] + list(np.cumsum(new)))
        x = normal(T, M)
        qkv = kernels.linear_w4(x, w_qkv)
        q, k, v = (t.view(T, -1, D) for t in qkv.split((H * D, KV * D, KV * D), 1))
        kernels.paged_append(cache, k, v, table, ints(lengths), starts)
        o = kernels.paged_attention_weighed(q, cache, weights, table, ints(lengths), starts)
        both = kernels.paged_attention_shared(q, cache, prefix, P, table, ints(lengths), starts)
        y = kernels.linear_w4(o.view(T, H * D), w_out, residual=x)
        # plain: what the cache holds, key by key
        held = lambda c, s, pages: (c[pages].float() * (torch.exp2(s[pages].float() - 127)[..., None, None] if eight else 1)).double()  # noqa: E731
        by_token = cache.values.view(torch.uint8 if eight else dtype).transpose(3, 4).reshape(cache.keys.shape).view(cache.keys.dtype)
        at = 0
        for b, (n, m) in enumerate(zip(lengths, new)):
            pages = table[b, :-(-n // page)].long()
            ks, vs = (held(c, s, pages).transpose(0, 1).reshape(KV, -1, D)[:, :n] for c, s in ((cache.keys, cache.key_scales), (by_token, cache.value_scales)))
            kp, vp = (held(c, s, prefix.long()).transpose(0, 1).reshape(KV, -1, D)[:, :150] for c, s in ((cache.keys, cache.key_scales), (by_token, cache.value_scales)))
            qq = q[at:at + m].double().transpose(0, 1)
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
            heads = lambda t: t.repeat_interleave(H // KV, 0)  # noqa: E731
            s = (qq @ heads(ks).transpose(1, 2)) * D ** -0.5
            for got, more_s, more_v in ((o, None, None), (both, (qq @ heads(kp).transpose(1, 2)) * D ** -0.5, heads(vp))):
                ss, vv = s.masked_fill(hidden, float("-inf")), heads(vs)
                if more_s is not None:
                    ss, vv = torch.cat((more_s, ss), 2), torch.cat((more_v, vv), 1)
                p = torch.softmax(ss, 2)
                u = torch.finfo(dtype).eps / 2
                bound = 1.01 * (u * (p @ vv).abs() + (u + 2.0 ** -13) * (p @ vv.abs())) + 2.0 ** -20
                assert ((got[at:at + m].double().transpose(0, 1) - p @ vv).abs() <= bound).all(), step
            at += m
        assert torch.isfinite(y).all()
        # as many rows' weights lie on the keys as there have been since the last eviction
        if step in (0, 3):
            left = kernels.paged_evict(cache, weights, table, ints(lengths), 30, 10)
            assert left.tolist() == [min(n, 40) for n in lengths]
            lengths = left.tolist()


@gpu
def test_refusals():
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([2] * 3, [30, 6, 0], 4, 2, 64, 16, torch.bfloat16, True)
    held, qd, w = cache.to_device(), q.cuda(), before.cuda()
    t, n, s = ints(table), ints(keys), ints(starts)
    assert kernels.paged_attention_weighed(qd[:0], held, w, t, n, s).shape == (0, 4, 64)
    assert torch.equal(w.cpu(), before)
    for args, error in [((qd, held, w.double(), t, n, s), TypeError), ((qd, held, w[1:], t, n, s), ValueError), ((qd, held, before, t, n, s), RuntimeError), ((qd[:, :3], held, w, t, n, s), ValueError),
                        ((qd.float(), held, w, t, n, s), TypeError), ((qd, held, w, t, n[:2], s), ValueError), ((qd, held, w, t.long(), n, s), TypeError), ((qd, held, w.transpose(1, 2), t, n, s), ValueError)]:
        with pytest.raises(error):
            kernels.paged_attention_weighed(*args)


def test_refusals_of_the_entry_point(lib):
    from tests.test_serving_host import Cache, Sequences
    base_c, base_s = dict(keys=16, values=16, ks=None, vs=None, pages=4, heads=2, page=16, D=32), dict(table=16, lengths=16, starts=16, B=2, width=3, T=5)

    def go(q=16, o=16, w=16, H=4, strides=True, dtype=3, work=16, size=1 << 30, c={}, s={}):
        st = (ctypes.c_int64 * 4)(128, 32, 128, 32) if strides is True else strides
        return lib.mhip_paged_attention_weighed(None, ctypes.byref(Cache(*{**base_c, **c}.values())), ctypes.byref(Sequences(*{**base_s, **s}.values())), q, o, w, H, 1.0, 1, st, dtype, work, size)

    assert go(q=None) == 1 and go(o=None) == 1 and go(w=None) == 1 and go(H=3) == 1 and go(strides=None) == 1 and go(work=None) == 1 and go(size=64) == 1 and go(s=dict(starts=None)) == 1
    assert go(dtype=1) == 2 and go(work=8) == 2 and go(strides=(ctypes.c_int64 * 4)(4, 32, 128, 32)) == 2 and go(c=dict(D=40)) == 2
    assert go(s=dict(T=0)) == 0 and go(s=dict(B=0)) == 0
