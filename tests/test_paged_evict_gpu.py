"""Eviction from a paged cache: which keys stay, in which order, and every bit of what moves, against a plain program over positions."""
import ctypes

import numpy as np
import pytest
import torch

from tests.paged_util import HostCache, table_of

gpu = pytest.mark.gpu
KINDS = pytest.mark.parametrize("eight,dtype", [(False, torch.bfloat16), (True, torch.bfloat16), (False, torch.float16)], ids=["bf16", "8bit", "f16"])
INTO = pytest.mark.parametrize("inplace", [False, True], ids=["into", "inplace"])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def stays(w, here, keep, recent):
    """Positions of a head that stay: w [n], here [n] whether a position has a page."""
    n = len(w)
    first = max(n - recent, 0)
    order = sorted((i for i in range(first) if here[i]), key=lambda i: (0, 0.0, i) if np.isnan(w[i]) else (1, -float(w[i]), i))
    return sorted(order[:keep]) + [i for i in range(first, n) if here[i]]


def e4m3(x):
    """Bytes of the e4m3 numbers nearest to x (ties to even) of |x| <= 448."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(np.where(x == 0, 1.0, x))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    r = np.abs(np.round(x / step) * step)
    _, e = np.frexp(np.where(r == 0, 1.0, r))
    normal = r >= 2.0 ** -6
    byte = np.where(normal, ((e - 1 + 7) << 3) + np.round((r / np.ldexp(1.0, e - 1) - 1) * 8).astype(int), np.round(r * 512).astype(int))
    return (byte | (np.signbit(x).astype(int) << 7)).astype(np.uint8)


class Plain:
    """A cache as arrays by token: keys and values [pages, KV, page, D] raw, scales, weights."""

    def __init__(self, held, weights):
        self.eight = held.key_scales is not None
        raw = lambda t: t.view(torch.uint8 if self.eight else torch.int16).cpu().numpy()  # noqa: E731
        self.k = raw(held.keys).copy()
        v = raw(held.values)
        self.v = v.transpose(0, 1, 2, 4, 3).reshape(self.k.shape).copy()
        self.scales = [s.cpu().numpy().astype(int) if s is not None else None for s in held[2:]]
        self.w = weights.cpu().numpy().copy()

    def evict(self, table, lengths, keep, recent, into):
        page, KV, pages = self.k.shape[2], self.k.shape[1], self.k.shape[0]
        left = []
        fresh = Plain.__new__(Plain)
        fresh.k, fresh.v, fresh.w, fresh.eight = self.k.copy(), self.v.copy(), self.w.copy(), self.eight
        fresh.scales = [s.copy() if s is not None else None for s in self.scales]
        to = table if into is None else into
        for b, n in enumerate(lengths):
            n = min(max(n, 0), table.shape[1] * page)
            here = [0 <= table[b, i // page] < pages for i in range(n)]
            count = 0
            for h in range(KV):
                w = np.array([self.w[table[b, i // page], h, i % page] if here[i] else 0 for i in range(n)], np.float32)
                src = stays(w, here, keep, recent)
                count = len(src)
                for j in range(0, len(src), page):
                    p, some = to[b, j // page], src[j:j + page]
                    if not 0 <= p < pages:
                        continue
                    for which, (a, out) in enumerate(((self.k, fresh.k), (self.v, fresh.v))):
                        x = np.stack([a[table[b, i // page], h, i % page] for i in some])
                        if self.eight:
                            was = np.array([self.scales[which][table[b, i // page], h] for i in some])
                            top = was.max()
                            value = torch.from_numpy(x).view(torch.float8_e4m3fn).double().numpy() * np.ldexp(1.0, np.maximum(was, 1) - max(top, 1))[:, None]
                            nan = np.isnan(value)
                            moved = np.where(nan, 0x7F, e4m3(np.where(nan, 0, value)))
                            x = np.where((np.maximum(was, 1) == max(top, 1))[:, None], x, moved)
                            fresh.scales[which][p, h] = top
                        out[p, h, :len(some)] = x
                    fresh.w[p, h, :len(some)] = [w[i] for i in some]
            left.append(count)
        self.__dict__.update(fresh.__dict__)
        return left


def same(plain, held, weights):
    now = Plain(held, weights)
    nan = lambda a: (a & 0x7F) == 0x7F if plain.eight else np.zeros(a.shape, bool)  # noqa: E731
    for a, b in ((plain.k, now.k), (plain.v, now.v)):
        assert ((a == b) | (nan(a) & nan(b))).all()
    for a, b in zip(plain.scales, now.scales):
        assert a is None or (a == b).all()
    assert np.array_equal(plain.w, now.w, equal_nan=True)


def make(lengths, KV, D, page, dtype, eight, seed=0, width=None, into_width=0, ties=False):
    rng = np.random.default_rng(seed)
    table, pages = table_of(lengths, page, rng, width)
    more = len(lengths) * into_width
    cache = HostCache(pages + more, KV, page, D, dtype, eight).fill(table, lengths, rng)
    held = cache.to_device()
    if eight:
        for s in held[2:]:                  # scales some powers of two apart, so that pages that come together round anew
            s.copy_((s.int() + torch.randint(-3, 4, s.shape, generator=torch.Generator().manual_seed(seed)).cuda()).clamp(1, 254).to(torch.uint8))
    w = rng.random((pages + more, KV, page), np.float32) ** 6
    if ties:
        w = np.round(w * 6).astype(np.float32)
    into = (pages + rng.permutation(more)).reshape(len(lengths), into_width) if into_width else None
    return held, torch.from_numpy(w).cuda(), np.asarray(table), into


def run(lengths, KV, D, page, dtype, eight, keep, recent, inplace, **kw):
    from metalhlo_amd import kernels
    most = max([min(n, keep + recent) for n in lengths] + [1])
    held, weights, table, into = make(lengths, KV, D, page, dtype, eight, into_width=0 if inplace else -(-min(keep + recent, max(kw.get("width") or 0, -(-max(lengths) // page)) * page) // page) or 1, **kw)
    plain = Plain(held, weights)
    want = plain.evict(table, lengths, keep, recent, into)
    got = kernels.paged_evict(held, weights, ints(table), ints(lengths), keep, recent, into=None if inplace else ints(into))
    assert got.tolist() == want and max(want) <= most
    same(plain, held, weights)


@gpu
@KINDS
@INTO
@pytest.mark.parametrize("D,page,KV", [(32, 16, 3), (64, 32, 2), (96, 64, 1), (128, 128, 2), (128, 256, 1), (64, 16, 1)])
def test_what_stays(D, page, KV, inplace, eight, dtype):
    run([300, 1, 0, 17, 64, 513, 129], KV, D, page, dtype, eight, 100, 20, inplace, seed=D + page)


@gpu
@INTO
@pytest.mark.parametrize("keep,recent", [(0, 0), (0, 1), (1, 0), (0, 40), (40, 0), (1, 1), (200, 0), (0, 200), (199, 1), (150, 50), (500, 500), (15, 1), (16, 16), (255, 1), (256, 0), (257, 0)])
def test_numbers_to_keep(keep, recent, inplace):
    run([200, 33, 400], 2, 32, 16, torch.bfloat16, True, keep, recent, inplace)


@gpu
@INTO
@pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
def test_equal_weights(eight, inplace):
    run([700, 90, 300], 2, 64, 32, torch.bfloat16, eight, 150, 7, inplace, ties=True)


@gpu
@INTO
def test_more_than_a_launch_holds_at_once(inplace):
    """Thousands of positions a head; more heads than units, which stay with one workgroup each where they lie."""
    run([9000, 20], 1, 32, 256, torch.bfloat16, True, 3000, 100, inplace)
    run([150 + 3 * b for b in range(40)], 8, 32, 16, torch.float16, False, 90, 10, inplace)


@gpu
@INTO
def test_weights_of_any_kind(inplace):
    from metalhlo_amd import kernels
    held, weights, table, into = make([400], 1, 64, 16, torch.bfloat16, False, into_width=0 if inplace else 8)
    flat = torch.zeros(400)
    flat[3], flat[5], flat[17], flat[100], flat[101], flat[390] = float("nan"), -1.0, float("inf"), float("-inf"), -0.0, 7.0
    flat[200:260] = torch.linspace(-3, 2, 60)
    flat[300:310] = 1e-42
    for i in range(400):
        weights[int(table[0, i // 16]), 0, i % 16] = flat[i]
    for keep, recent in ((2, 0), (60, 5), (120, 3)):
        w2, held2 = weights.clone(), type(held)(*(t.clone() if t is not None else None for t in held))
        plain = Plain(held2, w2)
        want = plain.evict(table, [400], keep, recent, into)
        got = kernels.paged_evict(held2, w2, ints(table), ints([400]), keep, recent, into=None if inplace else ints(into))
        assert got.tolist() == want
        same(plain, held2, w2)


@gpu
@INTO
@pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
def test_pages_that_are_none(eight, inplace):
    """Entries outside the cache hold no keys and take none; lengths beyond the table end with it."""
    from metalhlo_amd import kernels
    lengths = [300, 170, 5000, -4]
    held, weights, table, into = make([300, 170, 320, 1], 2, 64, 32, torch.bfloat16, eight, width=10, into_width=0 if inplace else 4)
    table[0, 8], table[2, 5], table[2, 9] = 1 << 30, -7, -1
    if not inplace:
        into[1, 1], into[2, 0] = -1, 1 << 20
    plain = Plain(held, weights)
    want = plain.evict(table, lengths, 90, 30, into)
    got = kernels.paged_evict(held, weights, ints(table), ints(lengths), 90, 30, into=None if inplace else ints(into))
    assert got.tolist() == want
    same(plain, held, weights)


@gpu
def test_shared_pages_are_left():
    """Sequences that share pages, each moved to its own."""
    from metalhlo_amd import kernels
    held, weights, table, into = make([320, 320], 2, 64, 32, torch.bfloat16, True, into_width=4)
    table[1, :6] = table[0, :6]
    plain = Plain(held, weights)
    want = plain.evict(table, [320, 310], 100, 20, into)
    assert kernels.paged_evict(held, weights, ints(table), ints([320, 310]), 100, 20, into=ints(into)).tolist() == want
    same(plain, held, weights)


@gpu
@pytest.mark.parametrize("many", [False, True])
def test_workspaces(many):
    """One for the list alone, a byte less than that, and one with room to gather; what lies behind its end stays."""
    from metalhlo_amd import _lib
    from tests.test_serving_host import Cache, Sequences
    lib, lengths = _lib.load(), ([90] * 300 if many else [300, 411])
    held, weights, table, _ = make(lengths, 1, 32, 16, torch.bfloat16, True)
    plain = Plain(held, weights)
    want = plain.evict(table, lengths, 50, 20, None)
    start = [t.clone() for t in (*held, weights)]
    c = Cache(*(t.data_ptr() for t in held), *held.keys.shape)
    t, n = ints(table), ints(lengths)
    s = Sequences(t.data_ptr(), n.data_ptr(), 0, len(lengths), t.shape[1], 0)
    least = ctypes.c_int64()
    need = lib.mhip_paged_evict_workspace(ctypes.byref(c), ctypes.byref(s), 50, 20, 1, ctypes.byref(least))
    assert need >= least.value > 0 and (need > least.value) == (not many)
    room = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    left = torch.empty(len(lengths), dtype=torch.int32, device="cuda")
    go = lambda size: lib.mhip_paged_evict(torch.cuda.current_stream().cuda_stream, ctypes.byref(c), ctypes.byref(s), weights.data_ptr(), 50, 20, None, 0, left.data_ptr(), room.data_ptr(), size)  # noqa: E731
    assert go(least.value - 1) == 1
    for size in {least.value, need - 1, need}:
        for a, b in zip((*held, weights), start):
            a.copy_(b)
        room.fill_(0xA5)
        assert go(size) == (1 if size < least.value else 0)
        if size >= least.value:
            assert left.tolist() == want
            same(plain, held, weights)
            assert (room[size:] == 0xA5).all()


@gpu
@INTO
def test_other_streams_and_graphs(inplace):
    from metalhlo_amd import kernels
    lengths = [300, 90, 200]
    held, weights, table, into = make(lengths, 2, 64, 32, torch.bfloat16, True, into_width=0 if inplace else 3)
    start = [t.clone() for t in (*held, weights)]
    args = (ints(table), ints(lengths), 60, 20, None if inplace else ints(into))
    plain = Plain(held, weights)
    want = plain.evict(table, lengths, 60, 20, into)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.paged_evict(held, weights, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert got.tolist() == want
    same(plain, held, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.paged_evict(held, weights, *args)
    for turn in range(3):
        for a, b in zip((*held, weights), start):
            a.copy_(b)
        weights.mul_(turn + 1.0)
        args[1][0] = 300 - 7 * turn
        plain = Plain(held, weights)
        want = plain.evict(table, [300 - 7 * turn, 90, 200], 60, 20, into)
        graph.replay()
        assert got.tolist() == want
        same(plain, held, weights)


@gpu
def test_none_at_all():
    from metalhlo_amd import kernels
    cache = kernels.paged_cache(4, 2, 16, 32, torch.bfloat16)
    weights = torch.zeros(4, 2, 16, device="cuda")
    assert kernels.paged_evict(cache, weights, ints(np.zeros((0, 3))), ints(np.zeros(0)), 5, 5).tolist() == []
    assert kernels.paged_evict(cache, weights, ints(np.zeros((2, 0))), ints([7, 0]), 5, 5).tolist() == [0, 0]


@gpu
def test_refusals():
    from metalhlo_amd import kernels
    held, weights, table, into = make([300, 90], 2, 64, 32, torch.bfloat16, True, into_width=3)
    t, n, i = ints(table), ints([300, 90]), ints(into)
    for args, error in [((held, weights, t, n, -1, 0), ValueError), ((held, weights, t, n, 0, -1), ValueError), ((held, weights, t, n, 97, 0, i), ValueError), ((held, weights.double(), t, n, 1, 1), TypeError),
                        ((held, weights[:, :1], t, n, 1, 1), ValueError), ((held, weights[:1], t, n, 1, 1), ValueError), ((held, weights, t.long(), n, 1, 1), TypeError), ((held, weights, t, n[:1], 1, 1), ValueError),
                        ((held, weights, t, n, 1, 1, i[:1]), ValueError), ((held, weights.cpu(), t, n, 1, 1), RuntimeError), ((held, weights, t, n, 1, 1, i.long()), TypeError),
                        ((held._replace(key_scales=None), weights, t, n, 1, 1), ValueError)]:
        with pytest.raises(error):
            kernels.paged_evict(*args)


def test_refusals_of_the_entry_point(lib):
    from tests.test_serving_host import Cache, Sequences
    base_c, base_s = dict(keys=16, values=16, ks=None, vs=None, pages=4, heads=2, page=16, D=32), dict(table=16, lengths=16, starts=None, B=2, width=3, T=0)

    def go(keep=5, recent=5, into=None, into_width=0, weights=16, left=16, work=16, size=1 << 20, c={}, s={}):
        return lib.mhip_paged_evict(None, ctypes.byref(Cache(*{**base_c, **c}.values())), ctypes.byref(Sequences(*{**base_s, **s}.values())), weights, keep, recent, into, into_width, left, work, size)

    assert go(keep=-1) == 1 and go(recent=-1) == 1 and go(into=16, into_width=0) == 1 and go(weights=None) == 1 and go(left=None) == 1 and go(work=None) == 1 and go(size=100) == 1
    assert go(c=dict(ks=16)) == 1 and go(c=dict(keys=None)) == 1 and go(s=dict(lengths=None)) == 1 and go(s=dict(table=None)) == 1 and go(s=dict(B=-1)) == 1
    assert go(c=dict(D=48)) == 2 and go(c=dict(page=24)) == 2 and go(work=8) == 2 and go(c=dict(keys=8)) == 2 and go(keep=1 << 31) == 2 and go(into=16, into_width=1 << 21) == 1
    assert go(s=dict(B=65536), c=dict(heads=1024, pages=1000)) == 2
    assert go(s=dict(B=0)) == 0
