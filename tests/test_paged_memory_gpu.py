"""What the operators on a cache in pages do at its ends: caches whose offsets pass 32 bits, sequences of more keys than a workgroup keeps at once, weights of any alignment, and no scratch memory."""
import os

import numpy as np
import pytest
import torch

from tests.test_paged_evict_gpu import INTO, run
from tests.test_paged_weighed_gpu import expected_weights, ints, make

gpu = pytest.mark.gpu
EIGHT = pytest.mark.parametrize("eight", [False, True], ids=["16bit", "8bit"])


@pytest.mark.parametrize("name", ["paged_join_kernel", "paged_weigh_kernel", "paged_add_kernel", "evict_select_kernel", "evict_move_kernel", "w4_rows_kernel", "w4_widen_kernel", "w4_quantize_kernel"])
def test_nothing_is_kept_in_scratch(name):
    pytest.importorskip("msgpack")
    from tests.test_kernel_resources import LIB, _kernels
    if not os.path.exists(LIB):
        pytest.skip("no built library")
    found = [k for k in _kernels() if name in k[".name"]]
    assert found
    assert [k[".name"] for k in found if k[".private_segment_fixed_size"] or k[".vgpr_spill_count"]] == []


@gpu
@INTO
@EIGHT
@pytest.mark.parametrize("n", [4096, 4097, 16385, 33000, 65536, 70001])
def test_sequences_of_many_keys(n, eight, inplace):
    """Weights in registers (4096, 16384, 32768 positions of what the table reaches), in LDS besides (65536), and read again."""
    run([n, 900], 1, 32, 256, torch.bfloat16, eight, 1500, 100, inplace, seed=n)


@gpu
@EIGHT
@pytest.mark.parametrize("off", [1, 2, 3, 4])
def test_weights_of_any_alignment(eight, off):
    from metalhlo_amd import kernels
    q, cache, table, keys, starts, before = make([1] * 5, [0, 61, 200, 1030, 15], 8, 2, 64, 32, torch.bfloat16, eight)
    room = torch.zeros(before.numel() + 8, device="cuda")
    weights = room[off:off + before.numel()].view(before.shape)
    weights.copy_(before)
    kernels.paged_attention_weighed(q.cuda(), cache.to_device(), weights, ints(table), ints(keys), ints(starts))
    want, bound = expected_weights(before, q, cache, table, keys, starts)
    assert (np.abs(weights.double().cpu().numpy() - want) <= bound).all()
    assert not room[:off].any() and not room[off + before.numel():].any()


@gpu
@EIGHT
@pytest.mark.parametrize("B,new", [(3, 1), (3, 70), (33, 1)])
def test_offsets_past_32_bits(B, new, eight):
    """The same pages at the end of a cache of 2^32 bytes and more: every result is the same, to the bit."""
    from metalhlo_amd import kernels
    KV, H, D, page = 8, 16, 128, 256
    dtype = torch.float8_e4m3fn if eight else torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(B + new)
    lengths = [(300, 700, 513, 257)[b % 4] for b in range(B)]
    counts = [-(-n // page) for n in lengths]
    few = sum(counts) + 3
    pages = (1 << 32) // (KV * page * D * (1 if eight else 2)) + few

    def cache_of(n):
        c = kernels.paged_cache(n, KV, page, D, dtype)
        return c, torch.empty(n, KV, page, device="cuda")

    small, w_small = cache_of(few)
    for x in small[:2]:
        x.copy_((torch.randn(x.shape, device="cuda", generator=gen)).to(dtype))
    if eight:
        for s in small[2:]:
            s.copy_(torch.randint(120, 128, s.shape, device="cuda", generator=gen).to(torch.uint8))
    w_small.copy_(torch.rand(w_small.shape, device="cuda", generator=gen))
    large, w_large = cache_of(pages)
    for a, b in zip((*small, w_small), (*large, w_large)):
        if a is not None:
            b[pages - few:].copy_(a)
    table, at = torch.full((B, max(counts)), -1, dtype=torch.int32), 3
    for b, n in enumerate(counts):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randn(B * new, H, D, device="cuda", generator=gen).to(torch.bfloat16)
    starts = ints(range(0, B * new + 1, new))
    results = []
    for cache, w, offset in ((small, w_small, 0), (large, w_large, pages - few)):
        t = torch.where(table >= 0, table + offset, table).cuda()
        shared = kernels.paged_attention_shared(q, cache, ints([offset, offset + 1, offset + 2]), ints([600]), t, ints(lengths), starts)
        out = kernels.paged_attention_weighed(q, cache, w, t, ints(lengths), starts)
        left = kernels.paged_evict(cache, w, t, ints(lengths), 150, 40)
        results.append([shared, out, left, w[offset:offset + few], *(x[offset:offset + few] for x in cache if x is not None)])
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)


@gpu
def test_numbers_to_keep_that_no_integer_adds_up():
    from metalhlo_amd import kernels
    cache = kernels.paged_cache(4, 1, 16, 32, torch.bfloat16)
    weights, table = torch.zeros(4, 1, 16, device="cuda"), ints([[0, 1]])
    for keep, recent in ((2 ** 62, 2 ** 62), (2 ** 63 - 1, 1), (1, 2 ** 63 - 1), (2 ** 30 + 1, 0)):
        for into in (None, ints([[2]]), ints([[2, 3]])):
            with pytest.raises((ValueError, RuntimeError)):
                kernels.paged_evict(cache, weights, table, ints([20]), keep, recent, into)
