"""Parity of token log probabilities, entropy and alternatives with float64: small and odd vocabularies, rows that begin off 16-byte boundaries, one row and many, equal values, rows in an order that
favours one group of lanes, masked, infinite and not-a-number logits."""
import numpy as np
import pytest
import torch

from tests.util import NAME

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda d: NAME[d])
STEP = 2.0 ** -24


def _check(x, tokens, top, what=""):
    """x [rows, vocab] on the device.  A lane of a workgroup of 256 adds n / 256 weights one after the other and the tree another few dozen, at 2 ** -24 each; a weight of exponent d is off by
    (4 + 2 |d|) 2 ** -24; the reference lies up to 8 below the maximum."""
    from metalhlo_amd import kernels
    got = kernels.token_log_probs(x, tokens, top=top)
    assert len(got) == (4 if top else 2) and all(t.dtype == torch.float32 for t in got[:3])
    d64 = x.double().cpu().numpy()
    rows, n = d64.shape
    t = tokens.cpu().numpy().astype(np.int64)
    with np.errstate(all="ignore"):
        m = d64.max(1, keepdims=True)
        d = d64 - m
        e = np.exp(d)
        total = e.sum(1, keepdims=True)
        log_p = d - np.log(total)
        p = e / total
        entropy = -np.where(e > 0, p * log_p, 0.0).sum(1)
        entropy[np.isnan(total[:, 0])] = np.nan
        far = np.where(e > 0, np.abs(d), 0.0) + 8
        mean = (p * far).sum(1)
        count = n / 256 + 64
        entropy_off = STEP * (count * (1 + mean) + (p * (4 + 2 * far) * (far + mean[:, None])).sum(1)) + 1e-7
        off = STEP * (count + 8 * np.abs(m) + 8 * np.abs(np.where(np.isfinite(log_p), log_p, 0.0)) + 8 * np.where(np.isfinite(d64), np.abs(d64), 0.0))
    inside = (t >= 0) & (t < n)
    at = np.where(inside, t, 0)
    want = np.where(inside, log_p[np.arange(rows), at], np.nan)

    def close(g, w, b):
        g = g.double().cpu().numpy()
        same = (g == w) | (np.isnan(g) & np.isnan(w))
        with np.errstate(invalid="ignore"):
            ok = same | (np.abs(g - w) <= b)
        assert ok.all(), (what, np.argwhere(~ok)[:4], g[~ok][:4], w[~ok][:4])
    close(got[0], want, off[np.arange(rows), at])
    close(got[1], entropy, entropy_off)
    if top:
        order = torch.sort(x.float().cpu(), dim=1, descending=True, stable=True).indices[:, :top].numpy()
        assert (got[3].cpu().numpy() == order).all(), (what, got[3].cpu().numpy()[:2, :8], order[:2, :8])
        close(got[2], np.take_along_axis(log_p, order, 1), np.take_along_axis(off, order, 1))
    return got


def _logits(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * scale).to(dtype).cuda(), torch.randint(0, vocab, (rows,), generator=g).int().cuda()


@TYPES
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (5, 64, 64), (2, 500, 50), (4, 2501, 64), (300, 777, 5), (3, 4096, 64), (7, 8191, 1), (2, 12345, 20), (1, 50257, 20),
                                            (130, 50257, 50), (600, 33000, 0), (3, 130001, 64)], ids=str)
def test_sizes(rows, vocab, top, dtype):
    _check(*_logits(rows, vocab, dtype, rows + vocab), top, str((rows, vocab, top)))


@TYPES
@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("vocab,top", [(5000, 64), (20001, 20)], ids=str)
def test_orders_of_a_row(rows, vocab, top, dtype):
    """Equal values go to the lowest index; a row that grows, one that falls, and one whose greatest values all lie in the pieces of a few groups of lanes."""
    i = torch.arange(vocab, device="cuda").float()
    per = 16 // torch.finfo(dtype).bits * 8
    some = ((i // per) % 512 < 8 * top) * 10.0 + (i % 97) / 50
    kinds = [torch.zeros(vocab, device="cuda"), i / vocab * 20, -i / vocab * 20, some, (i % 3), torch.where(i == vocab - 1, 5.0, -i * 0)]
    x = torch.stack([kinds[r % len(kinds)] for r in range(rows)]).to(dtype)
    _check(x, (torch.arange(rows, device="cuda") * 131 % vocab).int(), top)


@pytest.mark.parametrize("rows", [3, 600])
def test_more_candidates_than_are_kept(rows):
    """Every other group of lanes holds nothing but large values: thousands reach the bound."""
    vocab, top = 60000, 40
    i = torch.arange(vocab, device="cuda")
    x = torch.where(((i // 8) % 512 < 8 * 60)[None], torch.rand(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) + 9, 0.0).bfloat16()
    x[:, :vocab // 2][:, ::2] = 12.0
    _check(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), top)


@TYPES
@pytest.mark.parametrize("rows", [6, 640])
def test_masked_and_not_finite(rows, dtype):
    x, tokens = _logits(rows, 9001, dtype, 5)
    inf, nan = float("inf"), float("nan")
    x[0::6, ::2] = -inf
    x[1::6] = -inf
    x[2::6, 77] = inf
    x[3::6, 4444] = nan
    x[4::6] = -inf
    x[4::6, 8000] = 1.5
    x[5::6, 30:50], x[5::6, 9000] = nan, inf
    _check(x, tokens, 30)


def test_large_logits():
    x, tokens = _logits(4, 5000, torch.float32, 1)
    _check(x * 20 + 3000, tokens, 8)
    _check(x * 1e30, tokens, 8)
    _check(x * 1e-30, tokens, 8)


def test_tokens_outside_and_wide_ones():
    x, _ = _logits(5, 1000, torch.bfloat16)
    t = torch.tensor([-1, 0, 999, 1000, 1 << 40], device="cuda")
    got = _check(x, t, 3)
    assert torch.equal(torch.isnan(got[0]).cpu(), torch.tensor([True, False, False, True, True]))
    _check(x, t.clamp(max=2 ** 31 - 1).int(), 3)


@TYPES
def test_leading_axes_and_alignment(dtype):
    from metalhlo_amd import kernels
    x, t = _logits(6, 1001, dtype, 3)
    want = _check(x, t, 9)
    got = kernels.token_log_probs(x.view(2, 3, 1001), t.view(2, 3), top=9)
    assert [tuple(g.shape) for g in got] == [(2, 3), (2, 3), (2, 3, 9), (2, 3, 9)] and all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(got, want))
    for shift in (1, 3, 5):
        flat = torch.full((6 * 1001 + 16,), float("nan"), dtype=dtype, device="cuda")
        y = flat[shift:shift + 6006].view(6, 1001)
        y.copy_(x)
        _check(y, t, 9, f"shifted by {shift}")
    assert kernels.token_log_probs(x[0], t[0])[0].shape == () and kernels.token_log_probs(x[:0], t[:0], top=4)[2].shape == (0, 4)


def test_captured_and_on_another_stream():
    from metalhlo_amd import kernels
    x, t = _logits(3, 50257, torch.bfloat16, 9)
    buf, tok = x.clone(), t.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.token_log_probs(buf, tok, top=20)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = kernels.token_log_probs(buf, tok, top=20)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        y, u = _logits(3, 50257, torch.bfloat16, 20 + i)
        want = kernels.token_log_probs(y, u, top=20)
        buf.copy_(y)
        tok.copy_(u)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_refusals():
    from metalhlo_amd import _lib, kernels
    x, t = _logits(4, 100, torch.bfloat16)
    for call in (lambda: kernels.token_log_probs(x, t[:3]), lambda: kernels.token_log_probs(x, t, top=65), lambda: kernels.token_log_probs(x, t, top=-1),
                 lambda: kernels.token_log_probs(x[:, :4].contiguous(), t, top=5), lambda: kernels.token_log_probs(x[:, ::2], t), lambda: kernels.token_log_probs(x[:, :0], t)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.MhipError):
        kernels.token_log_probs(x.double(), t)
    with pytest.raises(_lib.MhipError):
        kernels.token_log_probs(x, t.short())
