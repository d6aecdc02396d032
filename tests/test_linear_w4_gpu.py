"""Linear layers with weights in 4 bits, and what makes them: against W = (q - zero) scale in 64 bits.

Bounds.  A group's products of q and x are exact and are added in fp32, then the groups: at most 128 + K / 128 + 16 additions of numbers whose magnitudes add up to
S = sum scale (q + zero) |x|, each wrong by half a step of 2^-24 of that at most.  The activation's slope is below 1.13 and its own error below 2^-20 of its argument.  Each rounding to 16 bits is half a step.
From 129 rows on W itself is rounded: half a step of every |w| |x| besides."""
import ctypes

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
ACT = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": torch.nn.functional.silu, "tanh": torch.tanh,
       "sigmoid": torch.sigmoid, "gelu_exact": torch.nn.functional.gelu}


def random_w4(N, K, group, dtype, seed=0, whole=True):
    """Words and scales as they lie in memory (anything in the words behind N and K), and (q, scale, zero) [N, K] in 64 bits."""
    rng = np.random.default_rng(seed)
    n16, k128 = -(-N // 16), -(-K // 128)
    q = rng.integers(0, 16, (n16 * 16, k128 * 128))
    zero = rng.integers(0, 16, (n16 * 16, k128 * 128 // group)).astype(np.float32)
    if not whole:
        zero = zero + rng.random(zero.shape, np.float32) * 0.9
    sz = torch.stack((torch.from_numpy(rng.uniform(0.5, 1.5, zero.shape).astype(np.float32) * 0.1), torch.from_numpy(zero)), -1).to(dtype)
    sz[N:] = 0
    sz[:, -(-K // group):] = 0
    # row 16 t + l % 16, column 128 b + 32 s + 8 (l / 16) + e; e in byte e % 4, its high half from 4 on
    v = q.reshape(n16, 16, k128, 4, 4, 8).transpose(0, 2, 4, 1, 3, 5).reshape(n16, k128, 64, 4, 8).astype(np.uint32)
    words = sum(v[..., e] << np.uint32(8 * (e % 4) + 4 * (e // 4)) for e in range(8)).astype(np.uint32)
    scales = sz.view(n16, 16, -1, 2).transpose(1, 2).contiguous()
    of = np.arange(K) // group
    return torch.from_numpy(words.view(np.int32)), scales, (torch.from_numpy(q[:N, :K]).double(), sz[:N, of, 0].double(), sz[:N, of, 1].double())


def expected(x, parts, bias=None, activation="none", residual=None):
    q, s, z = parts
    half, K = HALF[x.dtype], x.shape[-1]
    x64 = x.double().cpu().reshape(-1, K)
    y = x64 @ ((q - z) * s).t()
    err = (128 + K / 128 + 16) * 2.0 ** -24 * (x64.abs() @ ((q + z) * s).t())
    if x64.shape[0] >= 129:
        err = err + half * (x64.abs() @ ((q - z) * s).abs().t())
    if bias is not None:
        y = y + bias.double().cpu()
        err = err + 2.0 ** -24 * y.abs()
    if activation != "none":
        err = 1.13 * err + 2.0 ** -20 * y.abs() + 2.0 ** -22
    y = ACT[activation](y)
    err = err + half * (y.abs() + err) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)            # (f16's smallest numbers)
    if residual is not None:
        y = y + residual.double().cpu().reshape(y.shape)
        err = err + half * (y.abs() + err)
    return y, err


def check(got, x, parts, **more):
    want, err = expected(x, parts, **more)
    got = got.double().cpu().reshape(want.shape)
    # (a result that is half a step or more beyond the type's greatest number is an infinity: 65520 and more in float16, whose last step is 32)
    most = torch.finfo(x.dtype).max * (1 + HALF[x.dtype] / 2)
    beyond = want.abs() - err >= most
    assert (got[beyond] == torch.copysign(torch.tensor(float("inf"), dtype=torch.float64), want[beyond])).all()
    maybe = torch.isinf(got) & (want.abs() + err >= most)
    off = torch.where(beyond | maybe, 0.0, (got - want).abs())
    assert torch.isfinite(off).all() and (off <= err).all(), float((off / err).max())


def layer(words, scales, parts, group):
    from metalhlo_amd import kernels
    N, K = parts[0].shape
    return kernels.W4(words.cuda(), scales.cuda(), N, K, group)


def normal(shape, dtype, seed=1, std=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * std).to(dtype).cuda()


@gpu
@TYPES
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 300])
def test_rows(M, group, dtype):
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(272, 1408, group, dtype, M)
    x = normal((M, 1408), dtype)
    w = layer(words, scales, parts, group)
    got = kernels.linear_w4(x, w)
    check(got, x, parts)
    assert torch.equal(kernels.linear_w4(x, w), got)


@gpu
@TYPES
@pytest.mark.parametrize("K", [1, 7, 8, 31, 33, 100, 127, 128, 129, 136, 1000, 1001, 4104, 9000])
def test_columns_of_any_number(K, dtype):
    from metalhlo_amd import kernels
    for M, N, group in ((1, 40, 32), (3, 17, 64), (20, 16, 128), (50, 1, 32), (150, 33, 64)):
        words, scales, parts = random_w4(N, K, group, dtype, K)
        x = normal((M, K), dtype)
        bias, residual = normal((N,), dtype, 2), normal((M, N), dtype, 3)
        check(kernels.linear_w4(x, layer(words, scales, parts, group), bias, residual=residual), x, parts, bias=bias, residual=residual)


@gpu
@pytest.mark.parametrize("N", [1, 2, 3, 4, 6, 15, 16, 18, 31, 33, 1000, 5003])
def test_rows_of_weights_of_any_number(N):
    from metalhlo_amd import kernels
    for M, K, group in ((1, 256, 32), (16, 300, 128), (40, 520, 64), (131, 264, 32)):
        words, scales, parts = random_w4(N, K, group, torch.bfloat16, N)
        x = normal((M, K), torch.bfloat16)
        check(kernels.linear_w4(x, layer(words, scales, parts, group)), x, parts)


@gpu
@TYPES
@pytest.mark.parametrize("activation", list(ACT))
def test_activations(activation, dtype):
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(70, 500, 64, dtype)
    for M in (1, 30, 140):
        x, bias, residual = normal((M, 500), dtype, std=0.3), normal((70,), dtype, 2), normal((M, 70), dtype, 3)
        got = kernels.linear_w4(x, layer(words, scales, parts, 64), bias, activation, residual)
        check(got, x, parts, bias=bias, activation=activation, residual=residual)


@gpu
@TYPES
def test_zeros_between_whole_numbers(dtype):
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(64, 640, 32, dtype, whole=False)
    for M in (1, 64, 200):
        x = normal((M, 640), dtype)
        check(kernels.linear_w4(x, layer(words, scales, parts, 32)), x, parts)


@gpu
@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_tensors_off_sixteen_bytes(M):
    """x, bias and residual that begin at any element; leading axes."""
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(36, 264, 32, torch.bfloat16)
    w = layer(words, scales, parts, 32)
    for off in (1, 2, 4):
        x = normal((M * 264 + off,), torch.bfloat16)[off:].view(1, M, 264)
        bias, residual = normal((36 + off,), torch.bfloat16, 2)[off:], normal((M * 36 + off,), torch.bfloat16, 3)[off:].view(1, M, 36)
        got = kernels.linear_w4(x, w, bias, "silu", residual)
        assert got.shape == (1, M, 36)
        check(got, x, parts, bias=bias, activation="silu", residual=residual)


@gpu
def test_large_offsets_of_x():
    """Sums over x whose numbers share a large part, which the zeros take away again."""
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(48, 2048, 128, torch.float16)
    x = (normal((4, 2048), torch.float16) + 200).to(torch.float16)
    check(kernels.linear_w4(x, layer(words, scales, parts, 128)), x, parts)


@gpu
@pytest.mark.parametrize("M", [20, 140])
def test_what_is_not_finite_stays_in_its_row(M):
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(40, 300, 64, torch.bfloat16)
    w = layer(words, scales, parts, 64)
    x = normal((M, 300), torch.bfloat16)
    clean = kernels.linear_w4(x, w)
    x[3, 7], x[11, 299] = float("nan"), float("inf")
    got = kernels.linear_w4(x, w)
    rows = [r for r in range(M) if r not in (3, 11)]
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[11]).any() and torch.equal(got[rows], clean[rows])


@gpu
def test_no_rows_and_no_columns():
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(40, 300, 64, torch.bfloat16)
    assert kernels.linear_w4(torch.empty(0, 300, dtype=torch.bfloat16, device="cuda"), layer(words, scales, parts, 64)).shape == (0, 40)
    none = kernels.W4(torch.empty(0, 3, 64, 4, dtype=torch.int32, device="cuda"), torch.empty(0, 6, 16, 2, dtype=torch.bfloat16, device="cuda"), 0, 300, 64)
    assert kernels.linear_w4(normal((2, 300), torch.bfloat16), none).shape == (2, 0)
    assert kernels.quantize_w4(torch.empty(0, 5, device="cuda")).words.shape == (1, 0, 64, 4)


class Held(ctypes.Structure):
    _fields_ = [("words", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("N", ctypes.c_int64), ("K", ctypes.c_int64), ("group", ctypes.c_int64)]


@gpu
@pytest.mark.parametrize("M,K", [(129, 264), (200, 300), (300, 1001)])
def test_workspaces(M, K):
    """None, one that is a byte too small for the widened weights, and a whole one with anything in it; words behind its end stay."""
    from metalhlo_amd import _lib, kernels
    lib = _lib.load()
    words, scales, parts = random_w4(70, K, 32, torch.bfloat16)
    x, w = normal((M, K), torch.bfloat16), layer(words, scales, parts, 32)
    held = Held(w.words.data_ptr(), w.scales.data_ptr(), 70, K, 32)
    need = lib.mhip_linear_w4_workspace(M, ctypes.byref(held), kernels.DTYPE_CODE[x.dtype])
    assert need >= 70 * K * 2
    room = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    for size in (0, 70 * K * 2 - 1, need):
        out = torch.full((M * 70 + 16,), 7, dtype=torch.bfloat16, device="cuda")
        _lib.check(lib.mhip_linear_w4(torch.cuda.current_stream().cuda_stream, x.data_ptr(), ctypes.byref(held), None, None, out.data_ptr(), M, 0, kernels.DTYPE_CODE[x.dtype],
                                      room.data_ptr() if size else None, size))
        check(out[:M * 70].view(M, 70), x, parts)
        assert (out[M * 70:] == 7).all() and (room[max(size, 1):] == 0xA5).all() if size else True
    assert (room[need:] == 0xA5).all()


@gpu
@TYPES
@pytest.mark.parametrize("M,N,K,group", [(1, 40, 9000, 32), (4, 100, 5000, 128), (5, 300, 4100, 64), (24, 20, 20000, 128), (50, 200, 9000, 32), (100, 33, 7000, 64)])
def test_columns_dealt_over_the_device(M, N, K, group, dtype):
    """Few rows of a long K in parts: with the workspace, with a byte less of it, and with none; the same bits each time they are dealt."""
    from metalhlo_amd import _lib, kernels
    lib = _lib.load()
    words, scales, parts = random_w4(N, K, group, dtype)
    x, w, residual = normal((M, K), dtype), layer(words, scales, parts, group), normal((M, N), dtype, 3)
    held = Held(w.words.data_ptr(), w.scales.data_ptr(), N, K, group)
    need = lib.mhip_linear_w4_workspace(M, ctypes.byref(held), kernels.DTYPE_CODE[dtype])
    assert need > 0
    got = kernels.linear_w4(x, w, residual=residual)
    check(got, x, parts, residual=residual)
    room = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    for size in (0, need - 1, need):
        for turn in range(3):
            out = torch.full((M, N), 7, dtype=dtype, device="cuda")
            _lib.check(lib.mhip_linear_w4(torch.cuda.current_stream().cuda_stream, x.data_ptr(), ctypes.byref(held), None, residual.data_ptr(), out.data_ptr(), M, 0, kernels.DTYPE_CODE[dtype],
                                          room.data_ptr() if size else None, size))
            check(out, x, parts, residual=residual)
            assert size < need or torch.equal(out, got)
    assert (room[need:] == 0xA5).all()


@gpu
def test_other_streams_and_graphs():
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(100, 1500, 64, torch.float16)
    w = layer(words, scales, parts, 64)
    xs = {M: normal((M, 1500), torch.float16, M) for M in (1, 40, 150)}
    want = {M: kernels.linear_w4(x, w) for M, x in xs.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = {M: kernels.linear_w4(x, w) for M, x in xs.items()}
    torch.cuda.current_stream().wait_stream(side)
    for M in xs:
        assert torch.equal(there[M], want[M])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = {M: kernels.linear_w4(x, w) for M, x in xs.items()}
    for turn in range(3):
        for M, x in xs.items():
            x.copy_(normal((M, 1500), torch.float16, 10 * turn + M))
        graph.replay()
        for M, x in xs.items():
            assert torch.equal(got[M], kernels.linear_w4(x, w))


# ---- quantize_w4

def unpacked(w):
    """(q, scale, zero) [N16, K128] in 64 bits."""
    words = w.words.cpu().numpy().view(np.uint32)
    n16, k128 = words.shape[:2]
    q = np.stack([(words >> np.uint32(8 * (e % 4) + 4 * (e // 4))) & 15 for e in range(8)], -1).reshape(n16, k128, 4, 16, 4, 8).transpose(0, 3, 1, 4, 2, 5).reshape(n16 * 16, k128 * 128)
    sz = w.scales.double().cpu().transpose(1, 2).reshape(n16 * 16, -1, 2).repeat_interleave(w.group, 1)
    return torch.from_numpy(q.astype(np.float64)), sz[..., 0], sz[..., 1]


@gpu
@TYPES
@pytest.mark.parametrize("source", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,group", [(16, 128, 128), (5, 300, 32), (70, 1001, 64), (33, 31, 128)])
def test_quantize(N, K, group, source, dtype):
    """Every weight is held to half a step of its group's scale (its ends to what the rounding of the scale moves them besides: 15 steps times half a step of dtype), zeros exactly."""
    from metalhlo_amd import kernels
    rng = np.random.default_rng(N)
    m = torch.from_numpy((rng.standard_normal((N, K)) * np.exp(rng.standard_normal((N, 1)))).astype(np.float32)).to(source)
    m[:, 3::7] = 0
    if N > 4:
        m[1] = m[1].abs()                   # all of one sign
        m[2] = -0.25                        # all the same
        m[3] = 0
    views = {"[N, K]": (m.cuda(), True), "[K, N]": (m.t().contiguous().cuda(), False), "view": (torch.stack((m, -m), -1).cuda()[..., 0], True)}
    for name, (t, trans) in views.items():
        w = kernels.quantize_w4(t, group, dtype, trans_b=trans)
        assert (w.N, w.K, w.group) == (N, K, group)
        q, s, z = unpacked(w)
        assert (s[N:] == 0).all() and (z[N:] == 0).all() and (z == z.round()).all() and (z >= 0).all() and (z <= 15).all()
        held = ((q - z) * s)[:N, :K]
        want = m.double()
        assert ((held - want).abs() <= s[:N, :K] * (0.5 + 15 * HALF[dtype] + 2.0 ** -18) + (2.0 ** -25 * 15 if dtype == torch.float16 else 0)).all(), name
        assert (held[want == 0] == 0).all()
        span = torch.zeros(N, -(-K // group) * group, dtype=torch.float64)
        span[:, :K] = want
        span = span.view(N, -1, group)
        steps = (span.amax(2).clamp(min=0) - span.amin(2).clamp(max=0)) / 15
        assert ((s[:N].view(N, -1, group)[:, :steps.shape[1], 0] - steps).abs() <= HALF[dtype] * steps * 1.001 + 2.0 ** -25).all(), name
    x = normal((3, K), dtype)
    check(kernels.linear_w4(x, w), x, tuple(t[:N, :K] for t in (q, s, z)))


@gpu
def test_quantize_ends_of_range():
    from metalhlo_amd import kernels
    big = torch.tensor([[3.0e38, -3.0e38, 1.0e30] + [0.0] * 29], device="cuda")
    for dtype, most in ((torch.bfloat16, 3.3895313892515355e38), (torch.float16, 65504.0)):
        q, s, z = unpacked(kernels.quantize_w4(big, 32, dtype, trans_b=True))
        assert torch.isfinite(s).all() and s.max() <= most
    tiny = torch.full((1, 32), 1e-30, device="cuda")
    q, s, z = unpacked(kernels.quantize_w4(tiny, 32, torch.float16, trans_b=True))
    assert (s == 0).all() and (q == 0).all() and (z == 0).all()


@gpu
def test_refusals():
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(40, 300, 64, torch.bfloat16)
    w, x = layer(words, scales, parts, 64), normal((2, 300), torch.bfloat16)
    for call, error in [(lambda: kernels.linear_w4(x.float(), w), TypeError), (lambda: kernels.linear_w4(x.half(), w), TypeError), (lambda: kernels.linear_w4(x[:, :299], w), ValueError),
                        (lambda: kernels.linear_w4(x[:, :299].contiguous(), w), ValueError), (lambda: kernels.linear_w4(x.cpu(), w), RuntimeError),
                        (lambda: kernels.linear_w4(x, tuple(w)[:4]), TypeError), (lambda: kernels.linear_w4(x, w._replace(N=60)), ValueError), (lambda: kernels.linear_w4(x, w._replace(K=400)), ValueError),
                        (lambda: kernels.linear_w4(x, w._replace(group=16)), ValueError), (lambda: kernels.linear_w4(x, w._replace(group=128)), ValueError),
                        (lambda: kernels.linear_w4(x, w._replace(words=w.words.float())), ValueError), (lambda: kernels.linear_w4(x, w._replace(scales=w.scales.half())), TypeError),
                        (lambda: kernels.linear_w4(x, w, normal((41,), torch.bfloat16)), ValueError), (lambda: kernels.linear_w4(x, w, normal((40,), torch.float32)), TypeError),
                        (lambda: kernels.linear_w4(x, w, residual=normal((2, 41), torch.bfloat16)), ValueError), (lambda: kernels.linear_w4(x, w, activation="swish"), KeyError),
                        (lambda: kernels.quantize_w4(x[0]), ValueError), (lambda: kernels.quantize_w4(x, 48), ValueError), (lambda: kernels.quantize_w4(x, dtype=torch.float32), TypeError),
                        (lambda: kernels.quantize_w4(words.cuda()[0, 0]), Exception), (lambda: kernels.quantize_w4(x.cpu()), RuntimeError)]:
        with pytest.raises(error):
            call()


def test_refusals_of_the_entry_points(lib):
    """Sizes and pointers that are refused before anything is launched."""
    held = lambda **kw: ctypes.byref(Held(*{**dict(words=16, scales=16, N=32, K=128, group=32), **kw}.values()))  # noqa: E731
    go = lambda w, M=1, x=16, c=16, act=0, dtype=3, work=None: lib.mhip_linear_w4(None, x, w, None, None, c, M, act, dtype, work, 0)  # noqa: E731
    assert go(None) == 1 and go(held(N=-1)) == 1 and go(held(), M=-1) == 1 and go(held(), x=None) == 1 and go(held(), c=None) == 1 and go(held(words=None)) == 1 and go(held(), act=9) == 1
    assert go(held(group=48)) == 2 and go(held(), dtype=1) == 2 and go(held(words=8)) == 2 and go(held(), work=8) == 2 and go(held(K=0)) == 2 and go(held(N=1 << 25)) == 2 and go(held(), M=1 << 22) == 2
    assert go(held(), M=0) == 0 and go(held(N=0)) == 0
    quantize = lambda w, src=16, t=1, dtype=3: lib.mhip_quantize_w4(None, src, 1, 1, w, t, dtype)  # noqa: E731
    assert quantize(held(group=1)) == 2 and quantize(held(), t=7) == 2 and quantize(held(), src=None) == 1 and quantize(held(scales=None)) == 1 and quantize(held(scales=8)) == 2 and quantize(held(K=0)) == 0
    assert lib.mhip_linear_w4_workspace(500, held(N=-1), 3) == 0 and lib.mhip_linear_w4_workspace(500, None, 3) == 0


# ---- rows whose part of K is more than x's room in LDS

def wide_layer(N, K, group, dtype, seed):
    from metalhlo_amd import kernels
    n16, k128, g = -(-N // 16), -(-K // 128), torch.Generator(device="cuda").manual_seed(seed)
    words = torch.randint(-2 ** 31, 2 ** 31, (n16, k128, 64, 4), generator=g, device="cuda", dtype=torch.int32)
    scales = torch.empty(n16, k128 * (128 // group), 16, 2, device="cuda")
    scales[..., 0].uniform_(0.05, 0.15, generator=g)
    scales[..., 1] = torch.randint(0, 16, scales.shape[:3], generator=g, device="cuda")
    scales[:, -(-K // group):] = 0
    scales.view(n16, -1, 16, 2)[-1, :, N - 16 * (n16 - 1):] = 0
    return kernels.W4(words, scales.to(dtype), N, K, group)


def rows_of(w, tiles):
    """(q, scale, zero) [16 tiles, K] in 64 bits of those sixteens of rows."""
    from metalhlo_amd import kernels
    some = kernels.W4(w.words[tiles], w.scales[tiles], 16 * len(tiles), w.K, w.group)
    return tuple(t[:, :w.K] for t in unpacked(some))


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(28672, 8192), (12000, 8200), (12288, 12288), (11008, 16384), (8192, 28672)])
def test_few_rows_of_wide_layers(M, N, K, group):
    """One to five rows through layers that are long and wide, whose K few workgroups or none share."""
    from metalhlo_amd import kernels
    w = wide_layer(N, K, group, torch.bfloat16, K + M)
    x = normal((M, K), torch.bfloat16, M)
    got = kernels.linear_w4(x, w)
    tiles = [0, 1, N // 32, N // 16 - 1]
    parts = rows_of(w, tiles)
    check(got.view(M, N // 16, 16)[:, tiles].reshape(M, -1), x, parts)


@gpu
@TYPES
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K", [(1, 31000), (1, 40001), (2, 15873), (2, 33000), (3, 10625), (3, 20000), (4, 8065), (4, 9000), (4, 30001), (5, 20000)])
def test_few_rows_of_a_long_K_without_a_workspace(M, K, group, dtype):
    from metalhlo_amd import _lib, kernels
    w = wide_layer(48, K, group, dtype, K)
    x, out = normal((M, K), dtype), torch.full((M, 48), 7, dtype=dtype, device="cuda")
    held = Held(w.words.data_ptr(), w.scales.data_ptr(), 48, K, group)
    _lib.check(_lib.load().mhip_linear_w4(torch.cuda.current_stream().cuda_stream, x.data_ptr(), ctypes.byref(held), None, None, out.data_ptr(), M, 0, kernels.DTYPE_CODE[dtype], None, 0))
    check(out, x, rows_of(w, [0, 1, 2]))


# ---- infinities and great numbers.  A row whose sums of groups are not finite is added up weight by weight: K + 3 roundings at most of numbers whose magnitudes add up to S

def same_as_infinite(got, x, parts):
    """Rows in which W x holds infinities are these, NaN where they cancel or meet a weight of zero."""
    q, s, z = parts
    terms = ((q - z) * s)[None] * x.double().cpu()[:, None]                  # [rows, N, K]
    want = terms.sum(2)
    assert not torch.isfinite(want).any()
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])


@gpu
@TYPES
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 3, 16, 30, 100])
def test_infinities(M, group, dtype):
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(50, 1100, group, dtype, M, whole=group != 64)
    w = layer(words, scales, parts, group)
    x = normal((M, 1100), dtype, M)
    clean = kernels.linear_w4(x, w)
    rows = sorted({0, M // 2, M - 1})
    inf = float("inf")
    for places in ([(7, inf)], [(1099, -inf)], [(40, inf), (700, inf)], [(500, inf), (501, -inf)]):
        one = x.clone()
        for row in rows:
            for k, v in places:
                one[row, k] = v
        got, rest = kernels.linear_w4(one, w), [r for r in range(M) if r not in rows]
        same_as_infinite(got[rows], one[rows], parts)
        assert torch.equal(got[rest], clean[rest])
        bias, residual = normal((50,), dtype, 2), normal((M, 50), dtype, 3)
        both = kernels.linear_w4(one, w, bias, "relu", residual)[rows].float()
        plain = got[rows].float().relu() + residual[rows].float()
        assert torch.equal(both[got[rows] == inf], plain[got[rows] == inf]) and ((both - residual[rows].float())[got[rows] == -inf] == 0).all()
        one[rows[0], 3] = float("nan")
        assert torch.isnan(kernels.linear_w4(one, w)[rows[0]]).all()


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K", [(1, 264), (3, 4104), (12, 1000), (30, 264), (100, 1001)])
def test_great_numbers(M, K, group):
    """Groups whose sums of q x are beyond the greatest fp32 number, in results that are not."""
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(50, K, group, torch.bfloat16, M)
    scales = scales * torch.tensor([0.125, 1.0], dtype=torch.bfloat16)
    parts = (parts[0], parts[1] * 0.125, parts[2])
    w, x = layer(words, scales, parts, group), normal((M, K), torch.bfloat16)
    rows = sorted({0, M // 2, M - 1})
    for row in rows:
        for k, sign in ((0, 1), (3, 1), (9, -1), (17, 1), (30, 1), (K - 1, -1)):
            x[row, k] = sign * 2.0e38
    got = kernels.linear_w4(x, w)
    q, s, z = parts
    x64 = x.double().cpu()
    want, total = x64 @ ((q - z) * s).t(), x64.abs() @ ((q + z) * s).t()
    assert want.abs().max() > 1e37 and want.abs().max() < 3.2e38
    err = max(128 + K / 128 + 16, K + 3) * 2.0 ** -24 * total
    err = err + 2.0 ** -8 * (want.abs() + err)
    assert ((got.double().cpu() - want).abs() <= err).all()


@gpu
@pytest.mark.parametrize("group", [32, 128])
def test_as_many_rows_as_there_may_be(group):
    from metalhlo_amd import _lib, kernels
    M, K, N = 1 << 21, 40, 8
    words, scales, parts = random_w4(N, K, group, torch.float16)
    x, w = torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(0), device="cuda").half(), layer(words, scales, parts, group)
    out = torch.full((M, N), 7, dtype=torch.float16, device="cuda")
    held = Held(w.words.data_ptr(), w.scales.data_ptr(), N, K, group)
    _lib.check(_lib.load().mhip_linear_w4(torch.cuda.current_stream().cuda_stream, x.data_ptr(), ctypes.byref(held), None, None, out.data_ptr(), M, 0, kernels.DTYPE_CODE[x.dtype], None, 0))
    some = [0, 31, 32, 63, 64, M // 2, M - 65, M - 64, M - 33, M - 32, M - 1]
    check(out[some], x[some], parts)
    check(kernels.linear_w4(x, w)[-200:], x[-200:], parts)


@gpu
@TYPES
@pytest.mark.parametrize("M,K", [(129, 1100), (140, 1096), (300, 264)])
def test_infinities_of_many_rows(M, K, dtype):
    """From 129 rows on, with the widened W, as of few."""
    from metalhlo_amd import kernels
    words, scales, parts = random_w4(50, K, 64, dtype, M)
    w, x = layer(words, scales, parts, 64), normal((M, K), dtype, M)
    clean, inf, rows = kernels.linear_w4(x, w), float("inf"), [0, M // 2, M - 1]
    rest = [r for r in range(M) if r not in rows]
    for places in ([(7, inf)], [(K - 1, -inf)], [(40, inf), (K - 70, inf)], [(50, inf), (51, -inf)]):
        one = x.clone()
        for row in rows:
            for k, v in places:
                one[row, k] = v
        got = kernels.linear_w4(one, w)
        same_as_infinite(got[rows], one[rows], parts)
        assert torch.equal(got[rest], clean[rest])
