"""Parity of the operators on a paged cache against an oracle in float64: lengths around pages, blocks and tiles, head sizes and layouts, both forms of the cache, what lies
behind a sequence's end, pages that the table does not name, padded batches."""
import numpy as np
import pytest
import torch

from tests.paged_util import E4M3, HostCache, assert_within, attention, attention_at_once, half_step, scale_byte, table_of
from tests.util import NAME

pytestmark = pytest.mark.gpu
HALF = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda d: NAME[d])
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def _starts(new):
    return [0] + list(np.cumsum(new))


def _normal(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)


def _attend(lengths, new, H, KV, D, page, dtype, eight, causal=True, scale=None, pad=0, width=None, seed=0, change=None, spread=1.0, ahead=None):
    from metalhlo_amd import kernels
    rng = np.random.default_rng(seed)
    table, pages = table_of(lengths, page, rng, width)
    cache = HostCache(pages, KV, page, D, dtype, eight).fill(table, lengths, rng, spread)
    if change:
        change(table, cache)
    starts = _starts(new)
    q = _normal(rng, (starts[-1] + pad, H, D), dtype)
    held = cache.to_device()
    out = torch.full((starts[-1] + pad, H, D), 7.0, dtype=dtype, device="cuda")
    got = kernels.paged_attention(q.cuda(), held, ints(table), ints(lengths), ints(starts), scale=scale, is_causal=causal, out=out)
    assert got is out
    want, bound = attention(q, cache, table, lengths, starts, scale, causal)
    assert_within(got, want, bound, f"{lengths} {new} {(H, KV, D, page, eight, causal)}")
    assert (got[starts[-1]:] == 7).all()
    return got


@HALF
@EIGHT
@pytest.mark.parametrize("H,KV,D,page", [(1, 1, 64, 16), (12, 12, 64, 16), (8, 2, 128, 64), (6, 2, 96, 32), (5, 1, 32, 128), (32, 2, 128, 256)], ids=str)
def test_one_token(H, KV, D, page, dtype, eight):
    lengths = [1, 15, 16, 17, 63, 64, 65, 200, 257]
    _attend(lengths, [1] * len(lengths), H, KV, D, page, dtype, eight, seed=D + page)


@HALF
@EIGHT
@pytest.mark.parametrize("new", [[2, 1, 0, 5], [8, 3, 7, 4], [33, 1, 0, 70], [129, 128, 127, 1]], ids=str)
def test_several_tokens(new, dtype, eight):
    lengths = [n + c for n, c in zip(new, (0, 40, 30, 129))]
    _attend(lengths, new, 8, 4, 64, 16, dtype, eight, seed=len(new))


@EIGHT
@pytest.mark.parametrize("D,page", [(32, 32), (96, 64), (128, 128), (128, 16)], ids=str)
def test_pieces_of_prompts(D, page, eight):
    _attend([150, 300, 77], [150, 90, 40], 6, 2, D, page, torch.bfloat16, eight, seed=D)
    _attend([150, 300, 77], [150, 90, 40], 2, 2, D, page, torch.float16, eight, causal=False, scale=-0.2, seed=D)


@EIGHT
@pytest.mark.parametrize("new,H", [(1, 3), (1, 20), (50, 3)])
def test_long_caches_are_dealt_over_parts(new, H, eight):
    """Long next to short sequences: parts of unequal number, the last one short."""
    lengths = [9000, 3 + new, 2500, new, 70 + new]
    _attend(lengths, [new] * 5, H, 1, 64, 64, torch.bfloat16, eight, seed=new)


@EIGHT
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_without_keys(new, eight):
    """No keys at all, and fewer keys than new tokens: the rows in front of the first key yield zeros."""
    got = _attend([0, 5, new], [new, new + 3, new], 4, 2, 64, 16, torch.float16, eight, width=8)
    assert (got[:new] == 0).all()


@EIGHT
@pytest.mark.parametrize("new", [1, 45])
def test_pages_that_the_table_does_not_name(new, eight):
    def change(table, cache):
        table[0, 1], table[1, 0], table[2, :] = -1, 1 << 30, -7
        table[3, 2] = cache.x[0].shape[0]                           # the first one behind the cache
    got = _attend([100, 64, 80, 100], [new] * 4, 4, 2, 64, 32, torch.bfloat16, eight, causal=False, change=change)
    assert (got[2 * new:3 * new] == 0).all()


@EIGHT
def test_padded_batch_and_wide_table(eight):
    _attend([70, 33], [3, 1], 4, 2, 128, 16, torch.bfloat16, eight, pad=9, width=40)
    _attend([70, 133], [66, 100], 4, 2, 128, 16, torch.bfloat16, eight, pad=200, width=40)


def test_lengths_beyond_the_table_end_with_it():
    from metalhlo_amd import kernels
    rng = np.random.default_rng(3)
    table, pages = table_of([64], 16, rng)
    cache = HostCache(pages, 1, 16, 64, torch.bfloat16, False).fill(table, [64], rng)
    q = _normal(rng, (1, 1, 64), torch.bfloat16)
    held = cache.to_device()
    got = [kernels.paged_attention(q.cuda(), held, ints(table), ints([n]), ints([0, 1])) for n in (64, 65, 2 ** 31 - 1)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    assert (kernels.paged_attention(q.cuda(), held, ints(table), ints([-5]), ints([0, 1])) == 0).all()


@HALF
def test_large_scores(dtype):
    """Scores of some hundreds: one key takes all."""
    _attend([300, 40], [1, 1], 4, 4, 64, 16, dtype, False, scale=8.0, spread=3.0)
    _attend([300, 40], [100, 40], 4, 4, 64, 16, dtype, True, scale=8.0)


@EIGHT
@pytest.mark.parametrize("new", [1, 70])
def test_views_and_results_in_place(new, eight):
    from metalhlo_amd import kernels
    rng = np.random.default_rng(8)
    lengths, H, KV, D = [90, 71], 6, 3, 64
    table, pages = table_of(lengths, 16, rng)
    cache = HostCache(pages, KV, 16, D, torch.bfloat16, eight).fill(table, lengths, rng)
    held, starts = cache.to_device(), _starts([new, new])
    qkv = _normal(rng, (2 * new, (H + 2 * KV) * D), torch.bfloat16).cuda()
    q = qkv[:, :H * D].view(2 * new, H, D)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)          # heads outermost
    args = (held, ints(table), ints(lengths), ints(starts))
    want = kernels.paged_attention(q.contiguous(), *args)
    assert torch.equal(kernels.paged_attention(q, *args), want) and torch.equal(kernels.paged_attention(by_head, *args), want)
    kernels.paged_attention(q, *args, out=q)
    assert torch.equal(q, want)
    other = _normal(rng, (2 * new, (H + 2 * KV) * D), torch.bfloat16)
    assert torch.equal(kernels.paged_attention(by_head, *args, out=by_head), want) and other is not None


# ---------------------------------------------------------------- append
def _rope64(x, f):
    """x [n, heads, D], f [n, R] in float64, and the sum of the magnitudes that an element is formed of."""
    R = f.shape[1]
    h = R // 2
    y, size = x.copy(), np.abs(x)
    c, s = f[:, None, :h], f[:, None, h:]
    y[..., :h], y[..., h:R] = x[..., :h] * c - x[..., h:R] * s, x[..., :h] * s + x[..., h:R] * c
    size[..., :h] = np.abs(x[..., :h] * c) + np.abs(x[..., h:R] * s)
    size[..., h:R] = np.abs(x[..., :h] * s) + np.abs(x[..., h:R] * c)
    return y, size


def _append(lengths, new, H, KV, D, page, dtype, eight, R, positions=None, pad=0, seed=0, with_q=True, grow=1.0, change=None):
    """One append onto a cache that holds the older tokens, against the definition element by element."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(seed)
    table, pages = table_of(lengths, page, rng)
    old = [max(0, n - m) for n, m in zip(lengths, new)]
    cache = HostCache(pages, KV, page, D, dtype, eight, fill=3.0).fill(table, old, rng)
    if change:
        change(table)
    starts = _starts(new)
    T, P = starts[-1], positions if positions is not None else max(lengths)
    q, k, v = (_normal(rng, (T + pad, n, D), dtype) * grow for n in (H, KV, KV))
    freqs = None
    if R:
        angle = rng.uniform(-40, 40, (P, R // 2))
        freqs = torch.from_numpy(np.concatenate((np.cos(angle), np.sin(angle)), 1).astype(np.float32))
    held = cache.to_device()
    out = torch.full((T + pad, H, D), 5.0, dtype=dtype, device="cuda")
    got_q = kernels.paged_append(held, k.cuda(), v.cuda(), ints(table), ints(lengths), ints(starts), q=q.cuda() if R and with_q else None,
                                 freqs=freqs.cuda() if R else None, out=out if R and with_q else None)
    kd = held.keys.float().cpu().double().numpy()
    vd = held.values.float().cpu().double().transpose(3, 4).reshape(pages, KV, page, D).numpy()
    scales = [s.cpu().numpy() for s in held[2:]] if eight else None
    u, tiny = half_step(dtype), 2.0 ** -22                            # three fp32 roundings of a rotated element: 3 * 2 ** -24 of what it is formed of
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0            # f16 below 2 ** -14 has a step of 2 ** -24, half of which a rounding is off by
    expect = [x.double().numpy().copy() for x in cache.x]
    bound = [np.zeros_like(e) for e in expect]
    byte = [s.numpy().copy() for s in cache.scales] if eight else None
    for b, (n, m) in enumerate(zip(lengths, new)):
        pos = np.arange(n - m, n)
        ok = (pos >= 0) & ((pos < P) if R else True)
        rows = np.arange(starts[b], starts[b + 1])[ok]
        pos = pos[ok]
        if not len(pos):
            continue
        f = freqs.double().numpy()[pos] if R else np.zeros((len(pos), 0))
        kk, ks = _rope64(k.double().numpy()[rows], f)
        vv = v.double().numpy()[rows]
        if R and with_q:
            qq, qs = _rope64(q.double().numpy()[rows], f)
            g = got_q.double().cpu().numpy()[rows]
            assert (np.abs(g - qq) <= u * np.abs(qq) * 1.01 + tiny * qs + least).all()
        for at in np.unique(pos // page):
            p = table[b, at]
            if not 0 <= p < pages:
                continue
            mine = pos // page == at
            slot = pos[mine] % page
            for which, (x, size) in enumerate(((kk, ks), (vv, np.abs(vv)))):
                x, size = x[mine].transpose(1, 0, 2), size[mine].transpose(1, 0, 2)
                if not eight:
                    expect[which][p][:, slot] = x
                    bound[which][p][:, slot] = u * np.abs(x) * 1.01 + (tiny * size if which == 0 and R else 0) + least + 1e-30
                    continue
                for h in range(KV):
                    need = scale_byte(float(np.abs(x[h]).max()))
                    was = int(byte[which][p, h])
                    now = need if slot[0] == 0 else max(need, was)
                    if slot[0] and now > was:
                        moved = (torch.from_numpy(expect[which][p, h, :slot[0]]) * 2.0 ** (was - now)).float().to(E4M3).double().numpy()
                        expect[which][p, h, :slot[0]] = moved
                    byte[which][p, h] = now
                    y = x[h] * 2.0 ** (127 - now)
                    expect[which][p, h, slot] = y
                    # half a step of e4m3: 2 ** -4 of the value, 2 ** -10 below its normal numbers
                    bound[which][p, h, slot] = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10) * 1.0001 + tiny * size[h] * 2.0 ** (127 - now)
    for which, g in enumerate((kd, vd)):
        off = np.abs(g - expect[which])
        assert (off <= bound[which]).all(), (which, np.argwhere(off > bound[which])[:5], lengths, new)
        if eight:
            assert (scales[which] == byte[which]).all(), which
    if R and with_q:
        assert (got_q[T:] == 5).all()
    return held, got_q


@HALF
@EIGHT
@pytest.mark.parametrize("H,KV,D,page,R", [(12, 12, 64, 16, 0), (8, 2, 128, 64, 128), (6, 2, 96, 32, 48), (4, 1, 32, 128, 32), (8, 4, 128, 256, 64), (2, 1, 64, 16, 64)], ids=str)
def test_append(H, KV, D, page, R, dtype, eight):
    _append([1, 16, 17, 40, 300], [1, 1, 1, 40, 270], H, KV, D, page, dtype, eight, R, seed=D + page + R)
    _append([5, 0, 530, 33, 64], [5, 0, 3, 32, 1], H, KV, D, page, dtype, eight, R, seed=page, pad=3)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("grow", [1e-3, 1.0, 30.0, 2.0 ** 14])
def test_scales_grow_and_never_shrink(page, grow):
    """Tokens much smaller and much larger than those that a page holds: the held ones are rounded anew, down to nothing."""
    _append([page + 21, 9, 37], [3, 2, 17], 2, 2, 64, page, torch.bfloat16, True, 64, grow=grow, seed=page)


def test_a_page_begun_anew_forgets_its_scale():
    from metalhlo_amd import kernels
    c = kernels.paged_cache(1, 1, 16, 64, E4M3)
    c.key_scales.fill_(200)
    c.value_scales.fill_(255)
    x = torch.ones(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    kernels.paged_append(c, x, x * 500, ints([[0]]), ints([2]), ints([0, 2]))
    assert c.key_scales.item() == 119 and c.value_scales.item() == 128
    assert (c.keys.float()[0, 0, :2] == 256).all() and (c.values.float()[0, 0, 0, :, :2] == 256).all()      # 500 lies between 480 and 512 under the scale 2


def test_again_changes_nothing():
    held, q = _append([70, 33], [50, 2], 4, 2, 64, 32, torch.float16, True, 64, seed=4)
    again, q2 = _append([70, 33], [50, 2], 4, 2, 64, 32, torch.float16, True, 64, seed=4)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, again)) and torch.equal(q, q2)


@EIGHT
def test_tokens_without_a_place(eight):
    def change(table):
        table[0, 1], table[1, 0] = -1, 99
    _append([40, 10, 50], [40, 10, 3], 2, 2, 64, 16, torch.bfloat16, eight, 32, change=change)
    _append([3, 10], [8, 10], 2, 2, 64, 16, torch.bfloat16, eight, 32)                  # more tokens than keys
    _append([40, 10, 70], [40, 10, 70], 2, 2, 64, 32, torch.bfloat16, eight, 32, positions=37)


def test_what_is_not_finite():
    from metalhlo_amd import kernels
    c = kernels.paged_cache(1, 1, 16, 32, E4M3)
    x = torch.full((3, 1, 32), 2.0, dtype=torch.bfloat16, device="cuda")
    x[1, 0, 3], x[1, 0, 4], x[2, 0, 5] = float("inf"), float("nan"), float("-inf")
    kernels.paged_append(c, x, x, ints([[0]]), ints([3]), ints([0, 3]))
    assert c.key_scales.item() == c.value_scales.item() == 120
    for held in (c.keys.float()[0, 0, :3], c.values.float()[0, 0, 0].T[:3]):
        bad = ~torch.isfinite(x[:, 0].float())
        assert torch.isnan(held[bad]).all() and (held[~bad] == 256).all()


def test_views_and_turned_queries_in_place():
    from metalhlo_amd import kernels
    rng = np.random.default_rng(2)
    T, H, KV, D = 21, 6, 2, 64
    qkv = _normal(rng, (T, (H + 2 * KV) * D), torch.bfloat16).cuda()
    q, k, v = (t.view(T, -1, D) for t in qkv.split((H * D, KV * D, KV * D), 1))
    angle = torch.arange(64)[:, None] * torch.rand(32)
    freqs = torch.cat((angle.cos(), angle.sin()), 1).cuda()
    rest = (ints([[2, 0], [1, 3]]), ints([13, 30]), ints([0, 11, 21]))
    one, two = (kernels.paged_cache(4, KV, 16, D, E4M3) for _ in range(2))
    for c in (one, two):
        for t in c:
            t.view(torch.uint8).zero_()
    want = kernels.paged_append(one, k.contiguous(), v.contiguous(), *rest, q=q.contiguous(), freqs=freqs)
    kernels.paged_append(two, k, v, *rest, q=q, freqs=freqs, out=q)
    assert torch.equal(q, want) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, two))


# ---------------------------------------------------------------- both, as a program uses them
@EIGHT
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda d: NAME[d])
def test_steps_of_a_batch(dtype, eight):
    """Prompts, then tokens one by one: append and attend on the same tensors; in 16 bits the last rows are those of attention over everything at once."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(11)
    H, KV, D, page = 8, 2, 64, 16
    prompts, steps = [37, 1, 80], 5
    total = [n + steps for n in prompts]
    table, pages = table_of(total, page, rng)
    c = kernels.paged_cache(pages, KV, page, D, E4M3 if eight else dtype)
    x = [[_normal(rng, (n, h, D), dtype).cuda() for h in (H, KV, KV)] for n in total]
    done = [0, 0, 0]
    for step in range(steps + 1):
        new = prompts if step == 0 else [1, 1, 1]
        q, k, v = (torch.cat([x[b][j][done[b]:done[b] + new[b]] for b in range(3)]) for j in range(3))
        done = [a + b for a, b in zip(done, new)]
        args = (ints(table), ints(done), ints(_starts(new)))
        kernels.paged_append(c, k, v, *args)
        got = kernels.paged_attention(q, c, *args)
    for b in range(3):
        k, v = (x[b][j].repeat_interleave(H // KV, 1).double() for j in (1, 2))
        s = torch.einsum("hd,nhd->hn", x[b][0][-1].double().cpu(), k.cpu()) / 8
        p = torch.softmax(s, 1)
        want = torch.einsum("hn,nhd->hd", p, v.cpu())
        size = torch.einsum("hn,nhd->hd", p, v.abs().cpu())
        u = half_step(dtype)
        if eight:       # keys off by 2 ** -4 of themselves move a score by as much of |q| |k| / 8; values by 2 ** -4
            move = 2.0 ** -4 * torch.einsum("hd,nhd->hn", x[b][0][-1].double().abs().cpu(), k.abs().cpu()).max() / 8
            bound = (float(np.expm1(2 * float(move))) + 2.0 ** -4 + 2 * u) * size + 2.0 ** -4
        else:
            bound = 1.01 * (u * want.abs() + (u + 2.0 ** -13) * size) + 1e-4 * (dtype == torch.float16)
        assert ((got[b].double().cpu() - want).abs() <= bound).all()


def test_other_streams_and_graphs():
    """A step captured once and replayed for further tokens, which the tensors in device memory describe; two graphs share the pool; eager work between the replays."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(5)
    H, KV, D, page, B = 8, 2, 64, 16, 3
    start = [200, 31, 5000]
    table, pages = table_of([n + 8 for n in start], page, rng)
    cache = HostCache(pages, KV, page, D, torch.bfloat16, True).fill(table, start, rng)
    one, two = cache.to_device(), cache.to_device()
    table_d, starts = ints(table), ints([0, 1, 2, 3])
    tokens = [[_normal(rng, (B, h, D), torch.bfloat16).cuda() for h in (H, KV, KV)] for _ in range(6)]
    freqs = torch.randn(6000, 64, device="cuda")
    q, k, v = (t.clone() for t in tokens[0])
    lengths = ints([n + 1 for n in start])

    def step(c, q, k, v, lengths):
        turned = kernels.paged_append(c, k, v, table_d, lengths, starts, q=q, freqs=freqs)
        return kernels.paged_attention(turned, c, table_d, lengths, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    spare = cache.to_device()
    pool = torch.cuda.graph_pool_handle()
    with torch.cuda.stream(side):
        step(spare, q, k, v, lengths)
        for c in (one, spare):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side, pool=pool):
                got = step(c, q, k, v, lengths)
            graphs.append((g, got))
    torch.cuda.current_stream().wait_stream(side)
    for i, t in enumerate(tokens):
        for a, b in zip((q, k, v), t):
            a.copy_(b)
        want = step(two, *t, ints([n + 1 + i for n in start]))
        lengths.copy_(ints([n + 1 + i for n in start]))
        graphs[0][0].replay()
        first = graphs[0][1].clone()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want), i
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, two))


def test_refusals():
    from metalhlo_amd import _lib, kernels
    c = kernels.paged_cache(4, 2, 16, 64, torch.bfloat16)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, lengths, starts = ints([[0, 1]]), ints([3]), ints([0, 3])
    f = torch.zeros(32, 64, device="cuda")
    bad = [
        lambda: kernels.paged_append(c, k[:2], k, table, lengths, starts), lambda: kernels.paged_append(c, q, q, table, lengths, starts),
        lambda: kernels.paged_append(c, k, k.half(), table, lengths, starts), lambda: kernels.paged_append(c, k.half(), k.half(), table, lengths, starts),
        lambda: kernels.paged_append(c, k, k, table.long(), lengths, starts), lambda: kernels.paged_append(c, k, k, table, lengths, starts[:1]),
        lambda: kernels.paged_append(c, k, k, table, lengths, starts, q=q), lambda: kernels.paged_append(c, k, k, table, lengths, starts, q=q, freqs=f.half()),
        lambda: kernels.paged_append(c, k, k, table, lengths, starts, q=q[:2], freqs=f), lambda: kernels.paged_append(c, k, k, table, lengths, starts, out=q),
        lambda: kernels.paged_append(c, k, k, table, lengths, starts, freqs=torch.zeros(32, 80, device="cuda")),
        lambda: kernels.paged_append(c, k.transpose(1, 2), k, table, lengths, starts),
        lambda: kernels.paged_append(c, k, k, table, lengths, starts, q=q, freqs=f, out=q[:, :1].expand(3, 4, 64)),
        lambda: kernels.paged_attention(q[:, :3], c, table, lengths, starts), lambda: kernels.paged_attention(q.float(), c, table, lengths, starts),
        lambda: kernels.paged_attention(q[:, :, :32], c, table, lengths, starts), lambda: kernels.paged_attention(q, c, table, lengths[:0], starts),
        lambda: kernels.paged_attention(q, kernels.PagedCache(c.keys, c.keys), table, lengths, starts), lambda: kernels.paged_attention(q, c, table, lengths, starts, out=q[:, :2]),
        lambda: kernels.paged_attention(q, kernels.PagedCache(c.keys, c.values, ints([[0]])), table, lengths, starts),
        lambda: kernels.paged_attention(q, kernels.PagedCache(c.keys.view(torch.float8_e4m3fn), c.values.view(torch.float8_e4m3fn)), table, lengths, starts),
        lambda: kernels.paged_attention(q, c, table, lengths, starts, out=q[:, :1].expand(3, 4, 64)),
        lambda: kernels.paged_attention(q, c[:3], table, lengths, starts),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            raise AssertionError(i)
    flat = torch.zeros(3 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.MhipError, match="aligned"):
        kernels.paged_attention(flat[1:769].view(3, 4, 64), c, table, lengths, starts)
    with pytest.raises(_lib.MhipError, match="multiples of 8"):
        kernels.paged_attention(torch.zeros(3, 4 * 64 + 4, dtype=torch.bfloat16, device="cuda")[:, :256].view(3, 4, 64), c, table, lengths, starts)
    with pytest.raises(_lib.MhipError, match="multiple of 16"):
        kernels.paged_append(c, k, k, table, lengths, starts, freqs=torch.zeros(32, 24, device="cuda"))
    assert kernels.paged_attention(q[:0], c, table, lengths, starts).shape == (0, 4, 64)
    empty = ints(np.zeros((0, 2)))
    assert kernels.paged_append(c, k[:0], k[:0], empty, lengths[:0], starts[:1]) is None


@EIGHT
@HALF
@pytest.mark.parametrize("new,H", [(3, 4), (20, 4), (90, 2)])
def test_what_is_not_finite_stays_with_those_that_see_it(new, H, dtype, eight):
    """A NaN (and, in 16 bits, an infinity) among the values of new tokens: the tokens in front of them have finite results."""
    lengths, wild = [new + 70, new], {}

    def change(table, cache):
        for b, n in enumerate(lengths):
            for at, value, d in ((n - new // 2, float("nan"), 3), (n - 1, float("nan") if eight else float("inf"), 40), (n - 2, float("-inf") if not eight else float("nan"), 17)):
                cache.x[1][table[b, at // 16], :, at % 16, d] = value
                wild.setdefault(b, []).append((at, value, d))
    from metalhlo_amd import kernels
    rng = np.random.default_rng(new)
    table, pages = table_of(lengths, 16, rng)
    cache = HostCache(pages, 2, 16, 64, dtype, eight).fill(table, lengths, rng)
    starts = _starts([new, new])
    q = _normal(rng, (2 * new, H, 64), dtype)
    want, bound = attention(q, cache, table, lengths, starts)
    change(table, cache)
    got = kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(lengths), ints(starts)).double().cpu().numpy()
    for b, n in enumerate(lengths):
        for at, value, d in wild[b]:
            want[starts[b] + at - (n - new):starts[b + 1], :, d] += value
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    fine = np.isfinite(want)
    # (without the wild value the rows that see it are off in that element alone)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


@EIGHT
@pytest.mark.parametrize("lengths,context,H,KV,D,page", [([700, 1, 300, 900, 513], 0, 32, 32, 32, 16),            # more tiles than shares, short ones among them: whole tiles
                                                         ([300] * 40 + [5] * 60, 0, 8, 8, 32, 64),                  # the same with more than 64 sequences
                                                         ([130, 200, 90], 1500, 32, 8, 64, 32),                     # tiles split over shares
                                                         ([300] * 6, 900, 32, 32, 32, 256)], ids=str)               # more tiles than shares, all long
def test_many_tiles(lengths, context, H, KV, D, page, eight):
    from metalhlo_amd import kernels
    rng = np.random.default_rng(len(lengths))
    keys = [n + context for n in lengths]
    table, pages = table_of(keys, page, rng)
    cache = HostCache(pages, KV, page, D, torch.bfloat16, eight).fill(table, keys, rng)
    starts = _starts(lengths)
    q = _normal(rng, (starts[-1], H, D), torch.bfloat16)
    got = kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts))
    want, bound = attention_at_once(q, cache, table, keys, starts)
    assert_within(got, want, bound, "many tiles")
