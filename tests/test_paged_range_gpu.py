"""The operators on a paged cache at the ends of their types' ranges and of their tables: values and keys that float16 does not hold, scales far from one, sequences that are longer than their table, weights far
apart, many query heads to a key head; and attention over what an append has left in 8 bits, against what is held."""
import numpy as np
import pytest
import torch

from tests.paged_util import E4M3, HostCache, assert_within, attention, attention_at_once, half_step, table_of
from tests.util import NAME

pytestmark = pytest.mark.gpu
HALF = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda d: NAME[d])
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])
# tokens a sequence that put two query heads a key head into every form: 16 rows, 32 rows, tiles of 128, tiles of 256 (heads of 128 numbers in 16 bits)
NEW = pytest.mark.parametrize("new", [1, 3, 14, 90, 300])
ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731


def _batch(new, context, H, KV, D, page, dtype, eight, seed=0, width=None):
    rng = np.random.default_rng(seed)
    keys = [n + c for n, c in zip(new, context)]
    table, pages = table_of(keys, page, rng, width)
    cache = HostCache(pages, KV, page, D, dtype, eight).fill(table, keys, rng)
    starts = [0] + list(np.cumsum(new))
    q = torch.from_numpy(rng.standard_normal((starts[-1], H, D)).astype(np.float32)).to(dtype)
    return q, cache, table, keys, starts


def _attend(q, cache, table, keys, starts, **kw):
    from metalhlo_amd import kernels
    return kernels.paged_attention(q.cuda(), cache.to_device(), ints(table), ints(keys), ints(starts), **kw)


class Saturated(HostCache):
    """Values end at 65504, as float16 holds them."""

    def dense(self, which, table, b, n):
        x = super().dense(which, table, b, n)
        return np.clip(x, -65504.0, 65504.0) if which == 1 else x


def _rescale(cache, which, page, byte):
    """A page under another scale, its values rounded to it."""
    was = cache.scales[which][page].float()
    cache.x[which][page] = torch.nan_to_num(cache.x[which][page] * (2.0 ** (was - byte))[:, None, None]).to(E4M3).float()
    cache.scales[which][page] = byte


@NEW
@pytest.mark.parametrize("D", [64, 128])
def test_values_beyond_float16_end_there(new, D):
    """An 8-bit page whose largest value is float16's own holds 65536 = 256 * 2 ** 8 for it: the tokens that see it take 65504, those in front of it nothing of it."""
    q, cache, table, keys, starts = _batch([new, new], [40, 3], 4, 2, D, 16, torch.float16, True, seed=new)
    cache.__class__ = Saturated
    for b, n in enumerate(keys):
        p = table[b, (n - 1) // 16]
        _rescale(cache, 1, p, 135)
        cache.x[1][p, :, (n - 1) % 16, 5] = 256.0
        cache.x[1][p, :, (n - 1) % 16, 9] = -448.0              # (bfloat16 wrote it: 114688)
    got = _attend(q, cache, table, keys, starts)
    want, bound = attention(q, cache, table, keys, starts)
    assert_within(got, want, bound, f"{new}")


@NEW
def test_what_is_no_number_stays_one_beside_values_that_saturate(new):
    q, cache, table, keys, starts = _batch([new], [40], 4, 2, 64, 16, torch.float16, True, seed=new)
    cache.__class__ = Saturated
    n = keys[0]
    p = table[0, (n - 1) // 16]
    _rescale(cache, 1, p, 136)
    cache.x[1][p, :, (n - 1) % 16, 5] = 448.0
    want, bound = attention(q, cache, table, keys, starts)
    cache.x[1][p, :, (n - 1) % 16, 7] = float("nan")
    got = _attend(q, cache, table, keys, starts)
    assert torch.isnan(got[-1, :, 7]).all()
    got[-1, :, 7] = torch.from_numpy(want[-1, :, 7]).to(got)
    assert_within(got, want, bound, f"{new}")


@NEW
def test_keys_beyond_float16(new):
    """A key of 320 * 2 ** 8, which a rotation of float16's greatest numbers comes to: a row's score is what its product in fp32 is, whichever kernel serves it."""
    q, cache, table, keys, starts = _batch([new, new], [40, 3], 4, 2, 64, 16, torch.float16, True, seed=new)
    q = torch.where(q.abs() < 0.25, 0.25, q.float()).half()
    for b, n in enumerate(keys):
        p = table[b, (n - 1) // 16]
        _rescale(cache, 0, p, 135)
        cache.x[0][p, :, (n - 1) % 16] = 0.0
        cache.x[0][p, :, (n - 1) % 16, 11] = 320.0
    got = _attend(q, cache, table, keys, starts)
    want, bound = attention(q, cache, table, keys, starts)          # (scores of 81920 * |q| / 8, 2560 at least: the key has the whole weight, or none)
    assert_within(got, want, bound, f"{new}")


@HALF
@NEW
@pytest.mark.parametrize("by", [-40, 30])
def test_keys_whose_scales_are_far_from_one(by, new, dtype):
    """Keys of 2 ** by times the usual size under an attention scale that makes up for it."""
    q, cache, table, keys, starts = _batch([new, new], [40, 3], 4, 2, 64, 16, dtype, True, seed=new)
    cache.scales[0] = (cache.scales[0].int() + by).clamp(min=0).to(torch.uint8)
    scale = 2.0 ** (-by - 3)
    got = _attend(q, cache, table, keys, starts, scale=scale)
    want, bound = attention(q, cache, table, keys, starts, scale=scale)
    assert_within(got, want, bound, f"{by} {new}")


@NEW
@pytest.mark.parametrize("scale", [1e-35, 0.0, -1e-35])
def test_products_of_scales_that_are_no_float(scale, new):
    """A page's scale times the attention's is below every float: all keys alike, and masked ones none."""
    q, cache, table, keys, starts = _batch([new, new], [40, 3], 4, 2, 64, 16, torch.bfloat16, True, seed=new)
    cache.scales[0].fill_(3)
    got = _attend(q, cache, table, keys, starts, scale=scale)
    want, bound = attention(q, cache, table, keys, starts, scale=0.0)
    assert_within(got, want, bound, f"{scale} {new}")


@EIGHT
@NEW
@pytest.mark.parametrize("D", [64, 128])
def test_results_do_not_exceed_the_largest_value(new, D, eight):
    """Weights whose rounded sum is more than the sum they are divided by make more of float16's greatest number than it holds."""
    q, cache, table, keys, starts = _batch([new, new], [700, 90], 4, 2, D, 16, torch.float16, eight, seed=new)
    cache.__class__ = Saturated
    for p in table[table >= 0]:
        if eight:
            cache.scales[1][p] = 135
        cache.x[1][p] = 256.0 if eight else 65504.0
    got = _attend(q, cache, table, keys, starts, scale=0.3)
    want, bound = attention_at_once(q, cache, table, keys, starts, scale=0.3)
    assert bool(got.isfinite().all())
    assert_within(got, want, bound, f"{new}")


@HALF
@EIGHT
@NEW
def test_many_small_weights_beside_a_large_one(new, eight, dtype):
    """One key in 512 has weight 1, the others 2 ** -14.7, below float16's normal numbers: together they are a fiftieth and no rounding may lose them."""
    rng = np.random.default_rng(new)
    B, N, page, D = 2, 2048 + new, 64, 64
    table, pages = table_of([N] * B, page, rng)
    cache = HostCache(pages, 1, page, D, dtype, eight, fill=0.0)
    for b in range(B):
        for i in range(-(-N // page)):
            p = table[b, i]
            at = torch.arange(i * page, (i + 1) * page)
            cache.x[0][p, 0, :, 0] = torch.where(at % 512 == 3, 0.0, -1.0)
            cache.x[1][p, 0] = torch.where(at % 512 == 3, 1.0, 0.5)[:, None]
            if eight:
                cache.scales[0][p], cache.scales[1][p] = 127, 127
    starts = [0, new, 2 * new]
    q = torch.zeros(2 * new, 2, D, dtype=dtype)
    q[:, :, 0] = 10.1875                                      # exp(-10.1875) = 2 ** -14.7
    for causal in (False, True):
        got = _attend(q, cache, table, [N] * B, starts, scale=1.0, is_causal=causal)
        want, bound = attention_at_once(q, cache, table, [N] * B, starts, scale=1.0, is_causal=causal)
        assert_within(got, want, bound, f"{new} {causal}")


def test_bfloat16s_greatest_numbers_stay_finite():
    """An append rounds 3.38e38 to what a scale of 2 ** 120 has below 2 ** 128, half a step away at most."""
    from metalhlo_amd import kernels
    big = torch.finfo(torch.bfloat16).max
    for tokens in (1, 21):
        c = kernels.paged_cache(2, 2, 16, 64, E4M3)
        x = torch.full((tokens, 2, 64), big, dtype=torch.bfloat16, device="cuda")
        x[:, :, ::2] *= -1
        kernels.paged_append(c, x, x, ints([[0, 1]]), ints([tokens]), ints([0, tokens]))
        held = [c.keys.float()[0, :, :1].double() * 2.0 ** (c.key_scales[0].double() - 127)[:, None, None],
                c.values.float()[0, :, 0, :, :1].transpose(1, 2).double() * 2.0 ** (c.value_scales[0].double() - 127)[:, None, None]]
        for h in held:
            assert (h.abs() <= big).all() and ((h - x[0][:, None].double()).abs() <= 2.0 ** -4 * big).all()
        if tokens > 1:                                          # (a sum of these is beyond fp32)
            continue
        got = kernels.paged_attention(torch.zeros(tokens, 2, 64, dtype=torch.bfloat16, device="cuda"), c, ints([[0, 1]]), ints([tokens]), ints([0, tokens]))
        # one rounding of the result, and one of the weight
        assert ((got.double() - held[1].transpose(0, 1)).abs() <= 1.01 * 2 * half_step(torch.bfloat16) * big).all()


# ---------------------------------------------------------------- more keys than the table reaches
@EIGHT
@NEW
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_sequences_longer_than_their_table(causal, new, eight):
    """Keys behind a table's last column are keys that it does not name; the positions of the tokens are what the lengths say."""
    q, cache, table, keys, starts = _batch([new] * 3, [64 - new % 64 + 32, 300, 7], 4, 2, 64, 32, torch.bfloat16, eight, seed=new)
    for width in (1, 2, (new + 32) // 32, 5):
        short = table[:, :width].copy() if width < table.shape[1] else table
        padded = np.where(np.arange(table.shape[1])[None] < width, table, -1)
        got = _attend(q, cache, short, keys, starts, is_causal=causal)
        want, bound = attention(q, cache, padded, keys, starts, is_causal=causal)
        assert_within(got, want, bound, f"{width} {new} {causal}")


@EIGHT
@HALF
@pytest.mark.parametrize("lengths,new,width", [([35], [5], 2), ([33, 40, 7], [3, 9, 2], 2), ([17, 40, 16], [1, 1, 1], 1), ([33, 1000, 31], [1, 1, 1], 2), ([300, 16, 65], [200, 16, 65], 3),
                                               ([2000, 16, 48], [20, 16, 48], 3), ([9], [9], 0)], ids=str)
def test_append_to_sequences_longer_than_their_table(lengths, new, width, eight, dtype):
    """A token behind the table's last column takes no place, and no other's: the same as with columns that name no page."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(len(lengths))
    page, KV, H, D = 16, 2, 4, 64
    starts = [0] + list(np.cumsum(new))
    table = rng.permutation(3 * width + 1)[:len(lengths) * width].reshape(len(lengths), width)
    wide = -np.ones((len(lengths), 130), dtype=np.int32)
    wide[:, :width] = table
    k, v, q = (torch.from_numpy(rng.standard_normal((starts[-1], n, D)).astype(np.float32)).to(dtype).cuda() for n in (KV, KV, H))
    freqs = torch.from_numpy(rng.standard_normal((1990, 32)).astype(np.float32)).cuda()
    results = []
    for t in (table, wide):
        c = kernels.paged_cache(3 * width + 1, KV, page, D, E4M3 if eight else dtype)
        for held in c:
            if held is not None:
                held.view(torch.uint8).fill_(40)
        out = torch.full_like(q, 7)
        kernels.paged_append(c, k, v, ints(t), ints(lengths), ints(starts), q=q, freqs=freqs, out=out)
        results.append([out] + [held.view(torch.uint8) for held in c if held is not None])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@EIGHT
@pytest.mark.parametrize("new", [1, 40])
def test_freqs_without_positions(new, eight):
    """Every token lies outside of them: none is stored, and no query turned."""
    from metalhlo_amd import kernels
    c = kernels.paged_cache(8, 2, 16, 64, E4M3 if eight else torch.bfloat16)
    for held in c:
        if held is not None:
            held.view(torch.uint8).fill_(40)
    k, q = torch.ones(2 * new, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(2 * new, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 7)
    got = kernels.paged_append(c, k, k, ints(np.arange(8).reshape(2, 4)), ints([new + 3, new]), ints([0, new, 2 * new]), q=q, freqs=torch.empty(0, 32, device="cuda"), out=out)
    assert got is out and (out == 7).all() and all((held.view(torch.uint8) == 40).all() for held in c if held is not None)


# ---------------------------------------------------------------- both, as a program uses them
@HALF
@pytest.mark.parametrize("prompts,H,KV,D,page", [([37, 1, 80], 8, 2, 64, 16), ([300, 150, 33], 4, 2, 128, 64), ([20, 5, 16], 6, 3, 96, 32)], ids=str)
def test_attention_over_what_appends_have_left(prompts, H, KV, D, page, dtype):
    """Prompts, pieces behind them and single tokens onto an 8-bit cache; every step's attention against the bytes and scales that are held then."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(D)
    steps = [prompts, [1, 1, 1], [5, 0, 2], [1, 1, 1], [40, 3, 0], [1, 1, 1]]
    table, pages = table_of([sum(s[b] for s in steps) for b in range(3)], page, rng)
    c = kernels.paged_cache(pages, KV, page, D, E4M3)
    freqs = torch.from_numpy(rng.standard_normal((500, D)).astype(np.float32)).cuda()
    done = [0, 0, 0]
    for i, new in enumerate(steps):
        done = [a + b for a, b in zip(done, new)]
        starts = [0] + list(np.cumsum(new))
        q, k, v = (torch.from_numpy(rng.standard_normal((starts[-1], h, D)).astype(np.float32) * (1 + i)).to(dtype).cuda() for h in (H, KV, KV))
        args = (ints(table), ints(done), ints(starts))
        q = kernels.paged_append(c, k, v, *args, q=q, freqs=freqs)
        got = kernels.paged_attention(q, c, *args, scale=0.02)
        held = HostCache(pages, KV, page, D, dtype, True)
        held.x = [c.keys.float().cpu(), c.values.float().cpu().transpose(3, 4).reshape(pages, KV, page, D)]
        held.scales = [s.cpu() for s in c[2:]]
        want, bound = attention(q.cpu(), held, table, done, starts, scale=0.02)
        assert_within(got, want, bound, f"step {i}")


@EIGHT
@pytest.mark.parametrize("new,H", [(1, 40), (1, 200), (3, 200), (20, 300)])
def test_more_query_heads_to_a_key_head_than_a_tile_has_rows(new, H, eight):
    q, cache, table, keys, starts = _batch([new, new], [700, 2100], H, 1, 64, 16, torch.bfloat16, eight, seed=H)
    for causal in (True, False):
        got = _attend(q, cache, table, keys, starts, is_causal=causal)
        want, bound = attention_at_once(q, cache, table, keys, starts, is_causal=causal)
        assert_within(got, want, bound, f"{new} {H}")
