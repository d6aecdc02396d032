"""The operators of a serving step that is short of memory and of bytes a second, as cases that can be timed and compared:

  linear   a linear layer whose weights are held in 4 bits with a scale and a zero a group, for one token, a batch and a prompt
  shared   attention of a batch whose sequences have a long prefix in common and keys of their own behind it
  weighed  attention over a paged cache that adds up how much weight every key has been given
  evict    the keys of most weight and the latest ones move together, the others give their places back

`run` computes them in elementary torch operations in fp32, or with `own` by the calls of `metalhlo_amd.kernels`.  Both take the same memory:
a cache of keys [pages, heads, page, D] and values [pages, heads, page / 16, D, 16], in 16 bits or as e4m3 with a scale 2 ** (byte - 127) a page and head; weights of keys
[pages, heads, page] in fp32; 4-bit matrices [N, K] as words [N / 16, K / 128, 64, 4] (rounded up): lane l's word s holds row l % 16 of sixteen and the eight columns
from 32 s + 8 (l / 16) on, of which byte i has column i in its low four bits and column i + 4 in its high ones; scales [N / 16, K / group, 16, 2]: scale and zero of
w = (q - zero) * scale.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn


def _linear(rows, K, N, group, dtype="bf16", bias=False, activation="none", residual=False, **kw):
    return dict(kind="linear", rows=rows, K=K, N=N, group=group, dtype=dtype, bias=bias, activation=activation, residual=residual, **kw)


def _shared(B, new, prefix, context, H, KV, D, page, dtype="bf16", eight=True, uneven=0.5, **kw):
    return dict(kind="shared", B=B, new=new, prefix=prefix, context=context, H=H, KV=KV, D=D, page=page, dtype=dtype, eight=eight, uneven=uneven, **kw)


def _weighed(B, new, context, H, KV, D, page, dtype="bf16", eight=True, uneven=0.5, **kw):
    return dict(kind="weighed", B=B, new=new, prefix=0, context=context, H=H, KV=KV, D=D, page=page, dtype=dtype, eight=eight, uneven=uneven, **kw)


def _evict(B, context, keep, recent, KV, D, page, dtype="bf16", eight=True, uneven=0.5, inplace=False, **kw):
    return dict(kind="evict", B=B, new=0, prefix=0, context=context, keep=keep, recent=recent, H=KV, KV=KV, D=D, page=page, dtype=dtype, eight=eight, uneven=uneven, inplace=inplace, **kw)


def listed():
    return [
        # the projection in front of GPT-2's attention for one token: latency alone
        _linear(1, 768, 2304, 64, "f16", True, name="linear_one"),
        # one token through a wide layer: the weights' bytes
        _linear(1, 4096, 14336, 128, name="linear_step"),
        # a decode step of a batch, in front of a residual
        _linear(24, 5120, 5120, 128, residual=True, name="linear_batch"),
        # a prompt, with sizes that no tile divides
        _linear(1500, 4000, 4104, 64, "f16", True, "gelu", name="linear_prompt"),
        # a batch of conversations behind one long instruction, a token each
        _shared(64, 1, 12000, 400, 32, 8, 128, 64, uneven=0.9, name="shared_step"),
        # a few questions about one very long document
        _shared(6, 1, 100000, 900, 32, 8, 128, 256, name="shared_document"),
        # the questions themselves, behind a document of middle length, 16-bit cache
        _shared(12, 60, 6001, 0, 16, 4, 64, 32, "f16", False, uneven=0.6, name="shared_questions"),
        # one token of one conversation with GPT-2's heads
        _weighed(1, 1, 1000, 12, 12, 64, 16, "f16", name="weighed_one"),
        # a decode step of a batch
        _weighed(40, 1, 6000, 32, 8, 128, 64, uneven=0.6, name="weighed_step"),
        # whole prompts, whose tokens' weights begin with it
        _weighed(3, 1500, 0, 32, 8, 128, 64, "bf16", False, uneven=0.4, name="weighed_prompts"),
        # a batch whose caches are cut down to less than half
        _evict(32, 4000, 1500, 250, 8, 128, 64, uneven=0.3, name="evict_step"),
        # two long documents cut down where they lie, 16-bit cache
        _evict(2, 50000, 8000, 500, 8, 96, 32, "f16", False, inplace=True, name="evict_documents"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (max(hi, lo) / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "shared", "weighed", "evict"))
    half = rng.choice(("bf16", "bf16", "f16"))
    if kind == "linear":
        K, N = _log(rng, 100, 12000), _log(rng, 100, 14000)
        if rng.random() < 0.6:
            K, N = -(-K // 64) * 64, -(-N // 16) * 16
        rows = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 128), _log(rng, 129, 1500)))
        rows = max(1, min(rows, int(2.4e10 / (K * N))))
        return _linear(rows, K, N, rng.choice((32, 64, 128, 128)), half, rng.random() < 0.5, rng.choice(("none", "none", "gelu", "silu")), rng.random() < 0.3)
    D, KV = rng.choice((64, 128, 128, 96, 32)), rng.choice((1, 2, 4, 8, 12))
    H, page, eight = KV * rng.choice((1, 2, 4, 5, 8)), rng.choice((16, 32, 64, 128, 256)), rng.random() < 0.6
    uneven = round(rng.random() * 0.9, 2)
    if kind == "evict":
        context = _log(rng, 60, 30000)
        B = _log(rng, 1, max(1, min(48, 80_000_000 // (context * KV * D))))
        return _evict(B, context, max(1, int(context * rng.uniform(0.05, 0.9))), int(context * rng.uniform(0.0, 0.1)), KV, D, page, half, eight, uneven, rng.random() < 0.3)
    new = rng.choice((1, 1, _log(rng, 2, 12), _log(rng, 13, 400)))
    if kind == "shared":
        prefix, context = _log(rng, 100, 60000), rng.choice((0, _log(rng, 10, 1500)))
        prefix = max(1, min(prefix, int(1.5e11 / (4 * H * D * new))))
        B = _log(rng, 1, max(1, min(96, int(1.5e11 / (4 * H * D * new * (prefix + context))), 500_000_000 // (new * H * (prefix + context)))))
        return _shared(B, new, prefix, context, H, KV, D, page, half, eight, uneven)
    context = rng.choice((0, _log(rng, 16, 12000), _log(rng, 16, 12000)))
    B = _log(rng, 1, max(1, min(48, 50_000_000 // ((new + context) * H * max(D, new)))))
    return _weighed(B, new, context, H, KV, D, page, half, eight, uneven)


def _counts(c):
    """New tokens and own keys (the new ones included) of each sequence: up to `uneven` of them are missing."""
    lengths, new = [], []
    for i in range(c["B"]):
        less = c["uneven"] * ((i + 0.25) * 0.6180339887 % 1.0)
        n = max(1, c["new"] - int(c["new"] * less)) if c["new"] else 0
        new.append(n)
        lengths.append(n + c["context"] - int(c["context"] * (c["uneven"] * ((i + 0.75) * 0.7548776662 % 1.0))))
    return lengths, new


def _kept(c):
    return [min(n, c["keep"] + c["recent"]) for n in _counts(c)[0]]


def _power(e):
    """2 ** e in fp32 of whole e from -126 to 127 (a power that is computed may be off by a step, which breaks ties); 0 below."""
    return ((e.to(torch.int32) + 127).clamp(0, 254) << 23).view(torch.float32)


def _scaled(x, scale):
    """x as e4m3 at 2 ** (scale - 127)."""
    return (x * _power(127 - scale.to(torch.int32))).to(E4M3)


def _exponent_of(amax):
    """The byte of the least scale that holds amax within 448 = 1.75 * 2 ** 8."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.where(m > 0.875, e - 8, e - 9) + 127, torch.ones_like(e)).clamp(1, 254).to(torch.uint8)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    normal = lambda *shape, std=1.0, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)  # noqa: E731
    if c["kind"] == "linear":
        rows, K, N, group = c["rows"], c["K"], c["N"], c["group"]
        N16, K128 = -(-N // 16), -(-K // 128)
        packed = torch.randint(-2 ** 31, 2 ** 31, (N16, K128, 64, 4), generator=g, device="cuda", dtype=torch.int32)
        scales = torch.empty(N16, K128 * 128 // group, 16, 2, dtype=dt, device="cuda")
        scales[..., 0] = (torch.rand(scales.shape[:3], generator=g, device="cuda") + 0.5) * (0.2 * K ** -0.5)
        scales[..., 1] = (normal(*scales.shape[:3], std=1.5, dtype=torch.float32) + 7.5).round().clamp(0, 15)
        scales[:, -(-K // group):] = 0                           # behind the last column and the last row
        if N % 16:
            scales[-1, :, N % 16:] = 0
        return dict(case=c, x=normal(rows, K), packed=packed, scales=scales, bias=normal(N) if c["bias"] else None,
                    residual=normal(rows, N) if c["residual"] else None)

    lengths, new = _counts(c)
    B, H, KV, D, page, P = c["B"], c["H"], c["KV"], c["D"], c["page"], c["prefix"]
    T, width = sum(new), max(1, -(-max(lengths) // page))
    into_width = max(1, -(-max(_kept(c)) // page)) if c["kind"] == "evict" and not c["inplace"] else 0
    used = sum(-(-n // page) for n in lengths)
    pages = used + -(-P // page) + B * into_width + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table, at = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(lengths):
        table[b, :-(-n // page)] = order[at:at + -(-n // page)]
        at += -(-n // page)
    prefix = order[at:at + -(-P // page)].clone()
    at += -(-P // page)
    into = order[at:at + B * into_width].clone().view(B, into_width)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    # what the cache holds, the call's new tokens among it; where no token has been, whatever was in the memory
    held = E4M3 if c["eight"] else dt
    filled = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    inside = (torch.arange(width * page, device="cuda")[None] < as_int(lengths)[:, None]).view(B, width, page)
    filled[table[table >= 0].long()] = inside[table >= 0]
    if P:
        filled[prefix.long()] = (torch.arange(len(prefix) * page, device="cuda") < P).view(-1, page)

    def cache():
        x = normal(pages, KV, page, D)
        x.mul_(torch.rand(pages, KV, 1, 1, generator=g, device="cuda").add_(0.5).to(dt))
        scale = None
        if c["eight"]:
            scale = _exponent_of((x * filled[:, None, :, None]).abs().amax((2, 3)).float())
            x = _scaled(x.float(), scale[..., None, None]).view(torch.uint8)
        rest = torch.tensor(0x7F, dtype=torch.uint8, device="cuda") if c["eight"] else torch.tensor(float("nan"), dtype=dt, device="cuda")
        return torch.where(filled[:, None, :, None], x, rest).view(held), scale

    keys, key_scales = cache()
    values, value_scales = cache()
    values = values.view(torch.uint8 if c["eight"] else dt).view(pages, KV, page // 16, 16, D).transpose(3, 4).contiguous().view(held)
    state = dict(case=c, keys=keys, values=values, key_scales=key_scales, value_scales=value_scales, table=table, lengths=as_int(lengths), starts=as_int(starts),
                 most_new=max(new), most_keys=max(lengths))
    if c["kind"] != "evict":
        state["q"] = normal(T, (H + 2 * KV) * D)[:, :H * D].view(T, H, D)     # of the layer's projection
    if c["kind"] == "shared":
        state |= dict(prefix=prefix, prefix_length=as_int([P]))
    else:
        # weights that earlier steps have left: a few keys have most of them
        state["weights"] = torch.rand(pages, KV, page, generator=g, device="cuda").pow_(8.0).mul_(4.0) * filled[:, None]
    if c["kind"] == "evict":
        state |= dict(into=None if c["inplace"] else into, most_kept=max(_kept(c)))
    return state


# ---- the plain forms

def _plain_linear(s):
    c = s["case"]
    K, N, group = c["K"], c["N"], c["group"]
    w = s["packed"]
    N16, K128 = w.shape[:2]
    shifts = torch.tensor([0, 8, 16, 24, 4, 12, 20, 28], dtype=torch.int32, device="cuda")
    q = ((w[..., None] >> shifts) & 15).float()                                        # [N16, K128, 64, 4, 8]
    q = q.view(N16, K128, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(N16 * 16, K128 * 128 // group, group)
    sz = s["scales"].float().transpose(1, 2).reshape(N16 * 16, -1, 2)
    w = ((q - sz[..., 1:]) * sz[..., :1]).view(N16 * 16, K128 * 128)[:N, :K]
    y = torch.matmul(s["x"].float(), w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["activation"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    elif c["activation"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _by_token(values):
    """Values in blocks of sixteen tokens as [pages, KV, page, D], their bytes in 8 bits."""
    v = values.view(torch.uint8) if values.dtype == E4M3 else values
    return v.transpose(3, 4).reshape(v.shape[0], v.shape[1], v.shape[2] * 16, v.shape[3]).view(values.dtype)


def _held(cache, scales, pick):
    """[.., KV, keys, D] in fp32 of the pages pick [.., width]."""
    x = cache.view(torch.uint8)[pick].view(cache.dtype).float() if scales is not None else cache[pick].float()
    if scales is not None:
        x = x * _power(scales.to(torch.int32) - 127)[pick][..., None, None]
    x = x.transpose(-4, -3)
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], x.shape[-1])


def _own_scores(s):
    """Scores [B, KV, G, N, keys] of the sequences' own keys, the values [B, KV, keys, D] and where the tokens' rows lie among B * N."""
    c = s["case"]
    T, H, D = s["q"].shape
    KV, page, B = c["KV"], c["page"], c["B"]
    G, N = H // KV, s["most_new"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    row = torch.arange(T, device="cuda")
    b = (row[:, None] >= starts[None, 1:]).sum(1)
    place, p = b * N + row - starts[b], lengths[b] - (starts[b + 1] - row)
    pick = s["table"][:, :-(-s["most_keys"] // page)].long().clamp(min=0)
    at = torch.arange(pick.shape[1] * page, device="cuda")
    inside = (at[None] < lengths[:, None])[:, None, :, None]
    k = torch.where(inside, _held(s["keys"], s["key_scales"], pick), 0.0)
    v = torch.where(inside, _held(_by_token(s["values"]), s["value_scales"], pick), 0.0)
    q = torch.zeros(B * N, H, D, device="cuda").index_copy_(0, place, s["q"].float())
    q = q.view(B, N, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, D)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).view(B, KV, G, N, -1)
    sees = torch.full((B * N,), -1, dtype=torch.long, device="cuda").index_copy_(0, place, p).view(B, 1, 1, N, 1)
    x.masked_fill_(at > sees, float("-inf"))
    return x, v, place


def _rows(o, c, N, place):
    """[B, KV, G * N, D] -> the tokens' rows [T, H, D]."""
    B, KV, D = c["B"], c["KV"], c["D"]
    return o.view(B, KV, c["H"] // KV, N, D).permute(0, 3, 1, 2, 4).reshape(B * N, c["H"], D)[place]


def _plain_shared(s):
    c = s["case"]
    KV, D, N, P = c["KV"], c["D"], s["most_new"], c["prefix"]
    T, H, G = s["q"].shape[0], c["H"], c["H"] // c["KV"]
    # the prefix: the rows of all sequences at once
    pick = s["prefix"].long()
    k = _held(s["keys"], s["key_scales"], pick)[:, :P]
    v = _held(_by_token(s["values"]), s["value_scales"], pick)[:, :P]
    q = s["q"].float().view(T, KV, G, D).permute(1, 0, 2, 3).reshape(KV, T * G, D)
    y = torch.matmul(q, k.transpose(1, 2)).mul_(D ** -0.5)
    my = y.amax(-1, keepdim=True)
    y.sub_(my).exp_()
    oy, ly = torch.matmul(y, v), y.sum(-1, keepdim=True)
    back = lambda t: t.view(KV, T, G, -1).permute(1, 0, 2, 3).reshape(T, H, -1)  # noqa: E731
    my, ly, oy = back(my), back(ly), back(oy)
    # their own keys
    x, v, place = _own_scores(s)
    mx = x.amax(-1, keepdim=True)
    x.sub_(torch.where(mx > float("-inf"), mx, 0.0)).exp_()
    lx = x.sum(-1, keepdim=True)
    ox = torch.matmul(x.view(c["B"], KV, G * N, -1), v)
    rows = lambda t: t.reshape(c["B"], KV, G, N, -1).permute(0, 3, 1, 2, 4).reshape(c["B"] * N, H, -1)[place]  # noqa: E731
    mx, lx, ox = rows(mx), rows(lx), rows(ox)
    m = torch.maximum(mx, my)
    ax, ay = (mx - m).exp(), (my - m).exp()
    return ((ox * ax + oy * ay) / (lx * ax + ly * ay)).to(s["q"].dtype)


def _plain_weighed(s):
    c = s["case"]
    B, KV, page, N = c["B"], c["KV"], c["page"], s["most_new"]
    x, v, place = _own_scores(s)
    mx = x.amax(-1, keepdim=True)
    x.sub_(torch.where(mx > float("-inf"), mx, 0.0)).exp_()                            # (rows that are no tokens have no weights)
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total > 0, total, 1.0))
    given = x.sum((2, 3))                                                              # [B, KV, keys]
    o = _rows(torch.matmul(x.view(B, KV, -1, x.shape[-1]), v), c, N, place).to(s["q"].dtype)
    lengths, tokens = s["lengths"].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    at = torch.arange(x.shape[-1], device="cuda")
    b, key = torch.nonzero(at[None] < lengths[:, None], as_tuple=True)
    where, slot = s["table"].long()[b, key // page], key % page
    before = torch.where((key < (lengths - tokens)[b])[:, None], s["weights"][where, :, slot], 0.0)
    s["weights"][where, :, slot] = before + given[b, :, key]
    return o, s["weights"]


def _plain_evict(s):
    c = s["case"]
    B, KV, D, page, L, M = c["B"], c["KV"], c["D"], c["page"], s["most_keys"], s["most_kept"]
    lengths, table = s["lengths"].long(), s["table"].long()
    to = table if s["into"] is None else s["into"].long()
    at = torch.arange(L, device="cuda")
    inside = at[None] < lengths[:, None]
    pick = table.clamp(min=0)[:, at // page]                                           # [B, L]
    w = s["weights"][pick, :, (at % page)[None]].transpose(1, 2)                       # [B, KV, L]
    kept = torch.minimum(lengths, torch.full_like(lengths, c["keep"] + c["recent"]))
    # the last ones, and of the others as many of the greatest as there is room for
    late = inside & (at[None] >= (lengths - c["recent"])[:, None])
    rank = torch.sort(torch.where((inside & ~late)[:, None], w, float("-inf")), dim=2, descending=True, stable=True).indices
    order = torch.empty_like(rank).scatter_(2, rank, at.expand_as(rank).contiguous())
    stays = late[:, None] | ((inside & ~late)[:, None] & (order < c["keep"]))
    src = torch.sort(torch.where(stays, at, L), dim=2).values[:, :, :M]                 # [B, KV, M], L where there is none
    b, h, i = torch.nonzero(src < L, as_tuple=True)
    src = src[b, h, i]
    page_from, slot_from, page_to, slot_to = table[b, src // page], src % page, to[b, i // page], i % page
    s["weights"][page_to, h, slot_to] = s["weights"][page_from, h, slot_from]

    def move(cache, scales, by_token):
        if scales is None:
            by_token[page_to, h, slot_to] = by_token[page_from, h, slot_from]
            return by_token
        raw = by_token.view(torch.uint8)
        was = scales[page_from, h].int()
        grown = torch.full(scales.shape, -1, dtype=torch.int32, device="cuda").view(-1).scatter_reduce_(0, page_to * KV + h, was, "amax").view(scales.shape)
        x = (raw[page_from, h, slot_from].view(E4M3).float() * _power(was - grown[page_to, h])[:, None]).to(E4M3)
        raw[page_to, h, slot_to] = x.view(torch.uint8)
        scales.copy_(torch.where(grown >= 0, grown, scales.int()))
        return by_token

    move(s["keys"], s["key_scales"], s["keys"])
    kind = torch.uint8 if c["eight"] else s["values"].dtype
    pages, _, blocks = s["values"].shape[:3]
    moved = move(s["values"], s["value_scales"], _by_token(s["values"]).contiguous())
    s["values"].view(kind).copy_(moved.view(kind).view(pages, KV, blocks, 16, D).transpose(3, 4))
    return s["keys"], s["values"], s["key_scales"], s["value_scales"], s["weights"], kept.to(torch.int32)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"linear": _plain_linear, "shared": _plain_shared, "weighed": _plain_weighed, "evict": _plain_evict}[c["kind"]](s)
    from metalhlo_amd import kernels
    if c["kind"] == "linear":
        w = kernels.W4(s["packed"], s["scales"], c["N"], c["K"], c["group"])
        return kernels.linear_w4(s["x"], w, s["bias"], activation=c["activation"], residual=s["residual"])
    cache = kernels.PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"])
    if c["kind"] == "shared":
        return kernels.paged_attention_shared(s["q"], cache, s["prefix"], s["prefix_length"], s["table"], s["lengths"], s["starts"])
    if c["kind"] == "weighed":
        return kernels.paged_attention_weighed(s["q"], cache, s["weights"], s["table"], s["lengths"], s["starts"]), s["weights"]
    left = kernels.paged_evict(cache, s["weights"], s["table"], s["lengths"], c["keep"], c["recent"], into=s["into"])
    return s["keys"], s["values"], s["key_scales"], s["value_scales"], s["weights"], left


def work(case):
    c = case
    if c["kind"] == "linear":
        M, K, N = c["rows"], c["K"], c["N"]
        return dict(bytes=N * K / 2 + 4.0 * N * -(-K // c["group"]) + 2.0 * M * (K + N * (2 if c["residual"] else 1)) + (2.0 * N if c["bias"] else 0.0), flops=2.0 * M * N * K)
    lengths, new = _counts(c)
    T, H, KV, D, held = sum(new), c["H"], c["KV"], c["D"], 1 if c["eight"] else 2
    if c["kind"] == "evict":
        kept = sum(_kept(c))
        return dict(bytes=4.0 * KV * sum(lengths) + kept * KV * (4.0 * held * D + 4.0), flops=float(KV * sum(lengths)))
    pairs = sum(m * (n - m) + m * (m + 1) / 2 for n, m in zip(lengths, new)) + T * c["prefix"]
    told = 8.0 * KV * sum(lengths) if c["kind"] == "weighed" else 0.0
    return dict(bytes=4.0 * T * H * D + 2.0 * held * (c["prefix"] + sum(lengths)) * KV * D + told, flops=4.0 * pairs * H * D)


# ---- the definitions in 64 bits, row by row of pages and head by head

def _exact_linear(s):
    c = s["case"]
    N, K, group = c["N"], c["K"], c["group"]
    w = torch.zeros(s["packed"].shape[0], 16, s["packed"].shape[1] * 128, dtype=torch.float64, device="cuda")
    for quarter in range(4):
        for word in range(4):
            part = s["packed"][:, :, 16 * quarter:16 * quarter + 16, word]              # [N16, K128, 16]
            for e in range(8):
                w[:, :, 32 * word + 8 * quarter + e::128] = ((part >> (8 * (e % 4) + 4 * (e // 4))) & 15).double().transpose(1, 2)
    w = w.view(-1, w.shape[2])[:N, :K]
    sz = s["scales"].double().transpose(1, 2).reshape(-1, s["scales"].shape[1], 2)[:N]
    of = torch.arange(K, device="cuda") // group
    w = (w - sz[:, of, 1]) * sz[:, of, 0]
    y = s["x"].double() @ w.t()
    y = y if s["bias"] is None else y + s["bias"].double()
    if c["activation"] == "gelu":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    elif c["activation"] == "silu":
        y = torch.nn.functional.silu(y)
    return y if s["residual"] is None else y + s["residual"].double()


def _keys_of(s, pages, h, n):
    """Keys and values of a head in a row of pages, in 64 bits."""
    page, D = s["case"]["page"], s["case"]["D"]
    k = s["keys"][pages, h].double().reshape(-1, D)
    v = s["values"][pages, h].double().transpose(2, 3).reshape(-1, D)
    if s["case"]["eight"]:
        k = k * _power(s["key_scales"][pages, h].int() - 127).repeat_interleave(page)[:, None]
        v = v * _power(s["value_scales"][pages, h].int() - 127).repeat_interleave(page)[:, None]
    return k[:n], v[:n]


def _exact_attention(s):
    c = s["case"]
    lengths, new = _counts(c)
    KV, D, page, P = c["KV"], c["D"], c["page"], c["prefix"]
    G, out, at = c["H"] // KV, torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    weights = s["weights"].double() if c["kind"] == "weighed" else None
    for h in range(KV):
        if P:
            kp, vp = _keys_of(s, s["prefix"].long(), h, P)
        at = 0
        for b, (n, m) in enumerate(zip(lengths, new)):
            pages = s["table"][b, :-(-n // page)].long()
            k, v = _keys_of(s, pages, h, n)
            if P:
                k, v = torch.cat((kp, k)), torch.cat((vp, v))
            hidden = torch.arange(P + n, device="cuda")[None] > torch.arange(P + n - m, P + n, device="cuda")[:, None]
            given = torch.zeros(P + n, dtype=torch.float64, device="cuda")
            for j in range(h * G, h * G + G):
                w = torch.softmax((s["q"][at:at + m, j].double() @ k.t() / D ** 0.5).masked_fill(hidden, float("-inf")), 1)
                out[at:at + m, j] = w @ v
                given += w.sum(0)
            if weights is not None:
                old = weights[pages, h].reshape(-1)
                old[n - m:n] = 0.0
                old[:n] += given
                weights[pages, h] = old.view(-1, page)
            at += m
    return out if weights is None else (out, weights)


def _exact_evict(s):
    c = s["case"]
    lengths, _ = _counts(c)
    KV, D, page = c["KV"], c["D"], c["page"]
    keys, weights = s["keys"].double(), s["weights"].double()
    values = s["values"].double().permute(0, 1, 2, 4, 3).reshape(keys.shape).clone()
    for b, n in enumerate(lengths):
        total = min(n, c["keep"] + c["recent"])
        for h in range(KV):
            pages = s["table"][b, :-(-n // page)].long()
            w = weights[pages, h].reshape(-1)[:n]
            if total == n:
                src = torch.arange(n, device="cuda")
            else:
                first = n - c["recent"]
                best = torch.argsort(w[:first], descending=True, stable=True)[:c["keep"]]
                src = torch.cat((best.sort().values, torch.arange(first, n, device="cuda")))
            to = (s["table"] if s["into"] is None else s["into"])[b, :-(-total // page)].long()
            i = torch.arange(total, device="cuda")
            weights[to[i // page], h, i % page] = w[src]
            for cache, scales in ((keys, s["key_scales"]), (values, s["value_scales"])):
                x = cache[pages, h].reshape(-1, D)[src]
                if scales is not None:
                    e = scales[pages, h].long()[src // page]
                    top = torch.stack([e[j:j + page].max() for j in range(0, total, page)])[i // page]
                    x = x * _power(e - top)[:, None]
                    step = _power((torch.frexp(x).exponent - 1).clamp(min=-6) - 3)
                    x = torch.round(x / step) * step
                cache[to[i // page], h, i % page] = x
    values = values.view(*values.shape[:2], page // 16, 16, D).permute(0, 1, 2, 4, 3)
    return keys, values, None, None, weights, None


def exact(case, seed):
    if case["kind"] == "evict" and case["B"] * case["KV"] * max(_kept(case)) // case["page"] > 40000:
        return None
    s = prepare(case, seed)
    return _exact_linear(s) if case["kind"] == "linear" else _exact_evict(s) if case["kind"] == "evict" else _exact_attention(s)
