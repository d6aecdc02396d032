"""Rotation where a token's place in its sequence's pages is not its position: behind a prefix in common, and behind an eviction."""
import pytest
import torch

gpu = pytest.mark.gpu
KV, H, D, PAGE = 2, 4, 64, 16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def angles(positions):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    return torch.cat((a.cos(), a.sin()), 1).float().cuda()


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)


@gpu
@pytest.mark.parametrize("P", [1, 37, 160])
def test_behind_a_prefix(P):
    """Tokens appended with the rows of freqs from the prefix's length on are held as in one long sequence, and their attention is its."""
    from metalhlo_amd import kernels
    gen, n, freqs = torch.Generator("cuda").manual_seed(P), 50, angles(300)
    k, v, q = normal(gen, P + n, KV, D), normal(gen, P + n, KV, D), normal(gen, P + n, H, D)
    pages = -(-(P + n) // PAGE)
    one, two = (kernels.paged_cache(2 * pages + 2, KV, PAGE, D, torch.bfloat16) for _ in range(2))
    whole = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    turned = kernels.paged_append(one, k, v, whole, ints([P + n]), ints([0, P + n]), q=q, freqs=freqs)
    want = kernels.paged_attention(turned, one, whole, ints([P + n]), ints([0, P + n]))[P:]
    prefix, table = whole[0] + 1, (whole + 1 + pages).contiguous()
    kernels.paged_append(two, k[:P], v[:P], prefix[None], ints([P]), ints([0, P]), q=q[:P], freqs=freqs)
    own = kernels.paged_append(two, k[P:], v[P:], table, ints([n]), ints([0, n]), q=q[P:], freqs=freqs[P:])
    assert torch.equal(own, turned[P:])
    row = lambda cache, table, i: cache.keys[int(table[i // PAGE]), :, i % PAGE]  # noqa: E731
    assert all(torch.equal(row(two, prefix, i) if i < P else row(two, table[0], i - P), row(one, whole[0], i)) for i in range(P + n))
    got = kernels.paged_attention_shared(own, two, prefix, ints([P]), table, ints([n]), ints([0, n]))
    # (either is off by a rounding of its result and one of each weight, half a step of 2^-8)
    u = 2.0 ** -8
    assert ((got - want).double().abs() <= 2 * (u * want.double().abs() + (u + 2.0 ** -13) * 1.01 * v.double().abs().max())).all()


@gpu
def test_behind_an_eviction():
    """Tokens turned by their own positions and appended without freqs lie behind what is left, turned so."""
    from metalhlo_amd import kernels
    gen, freqs, lengths = torch.Generator("cuda").manual_seed(3), angles(300), [60, 100]
    cache = kernels.paged_cache(16, KV, PAGE, D, torch.bfloat16)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    kernels.paged_append(cache, normal(gen, 160, KV, D), normal(gen, 160, KV, D), table, ints(lengths), ints([0, 60, 160]), freqs=freqs)
    weights = torch.rand(16, KV, PAGE, generator=gen, device="cuda")
    left = kernels.paged_evict(cache, weights, table, ints(lengths), 20, 10)
    assert left.tolist() == [30, 30]
    q, k, v, positions = normal(gen, 2, H, D), normal(gen, 2, KV, D), normal(gen, 2, KV, D), torch.tensor(lengths, device="cuda")
    own = freqs[positions].to(k.dtype)
    qt, kt = (kernels.rope(t.transpose(0, 1).contiguous(), own).transpose(0, 1) for t in (q, k))
    kernels.paged_append(cache, kt, v, table, left + 1, ints([0, 1, 2]))
    x1, x2 = k.double().split(D // 2, 2)
    c, s = freqs[positions].double()[:, None].split(D // 2, 2)
    want, terms = torch.cat((x1 * c - x2 * s, x1 * s + x2 * c), 2), torch.cat(((x1 * c).abs() + (x2 * s).abs(), (x1 * s).abs() + (x2 * c).abs()), 2)
    held = torch.stack([cache.keys[int(table[b, 30 // PAGE]), :, 30 % PAGE] for b in range(2)]).double()
    # (cosines and sines of 16 bits, and the result's own rounding)
    assert ((held - want).abs() <= 1.01 * 2.0 ** -8 * (terms + want.abs())).all()
    o = kernels.paged_attention_weighed(qt, cache, weights, table, left + 1, ints([0, 1, 2]))
    keys = torch.stack([cache.keys[table[b, :2].long()].transpose(0, 1).reshape(KV, -1, D)[:, :31] for b in range(2)]).double().repeat_interleave(H // KV, 1)
    values = torch.stack([cache.values[table[b, :2].long()].transpose(3, 4).transpose(0, 1).reshape(KV, -1, D)[:, :31] for b in range(2)]).double().repeat_interleave(H // KV, 1)
    p = torch.softmax((keys @ qt.double()[..., None])[..., 0] * D ** -0.5, 2)
    full, total = (p[..., None] * values).sum(2), (p[..., None] * values.abs()).sum(2)
    assert ((o.double() - full).abs() <= 1.01 * (2.0 ** -8 * full.abs() + (2.0 ** -8 + 2.0 ** -13) * total) + 2.0 ** -20).all()
