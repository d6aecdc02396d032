"""The operators of a serving step that keeps its keys and values in pages, as cases that can be timed and compared:

  append   keys and values of new tokens into a paged cache, rotated on the way, in 16 bits or in 8 with a scale a page and head
  attend   attention over such a cache: decode steps, several tokens a sequence, prompts behind a context
  score    log probabilities of given tokens, the distribution's entropy and its top alternatives

`run` computes them in elementary torch operations in fp32, or with `own` by the calls of `metalhlo_amd.kernels`.  Both write the same cache:
keys [pages, heads, page, D] and values [pages, heads, page / 16, D, 16]; 8 bits are e4m3 with a scale 2 ** (byte - 127) a page and head.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
E4M3 = torch.float8_e4m3fn


def _append(B, new, context, H, KV, D, page, rotated, dtype="bf16", eight=True, uneven=0.5, **kw):
    return dict(kind="append", B=B, new=new, context=context, H=H, KV=KV, D=D, page=page, rotated=rotated, dtype=dtype, eight=eight, uneven=uneven, **kw)


def _attend(B, new, context, H, KV, D, page, dtype="bf16", eight=True, uneven=0.5, **kw):
    return dict(kind="attend", B=B, new=new, context=context, H=H, KV=KV, D=D, page=page, dtype=dtype, eight=eight, uneven=uneven, **kw)


def _score(rows, vocab, top, dtype="bf16", **kw):
    return dict(kind="score", rows=rows, vocab=vocab, top=top, dtype=dtype, **kw)


def listed():
    return [
        # one token of one conversation with GPT-2's heads, which have no rotation: latency alone
        _append(1, 1, 700, 12, 12, 64, 16, 0, "f16", name="append_one"),
        # a decode step of a batch: queries and keys rotated, a page's scale may grow
        _append(48, 1, 4000, 32, 8, 128, 64, 128, name="append_step"),
        # prompts of unequal length, the last page of each left open
        _append(5, 2600, 0, 32, 8, 128, 64, 128, uneven=0.7, name="append_prompts"),
        # a cache in 16 bits, half of each head rotated
        _append(7, 900, 333, 16, 16, 96, 32, 48, "bf16", False, name="append_16bit"),
        # one token of one conversation, GPT-2's heads
        _attend(1, 1, 1000, 12, 12, 64, 16, "f16", name="attend_one"),
        # a decode step of a batch whose contexts differ by a factor of five
        _attend(48, 1, 8000, 32, 8, 128, 64, uneven=0.8, name="attend_step"),
        # two long documents, four query heads to a key head
        _attend(2, 1, 120000, 32, 8, 128, 256, uneven=0.2, name="attend_long"),
        # a few tokens a sequence to be verified at once, 16-bit cache
        _attend(16, 5, 3001, 24, 8, 64, 32, "f16", False, name="attend_verify"),
        # the next pieces of three prompts behind what the cache holds of them
        _attend(3, 1024, 7001, 32, 8, 128, 64, uneven=0.6, name="attend_pieces"),
        # the distribution behind one token of a few conversations (GPT-2's vocabulary)
        _score(3, 50257, 20, name="score_step"),
        # the tokens of a prompt scored at once, fp32 logits
        _score(300, 32003, 5, "f32", name="score_f32"),
        # a batch of documents scored
        _score(4096, 50257, 20, name="score_documents"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("append", "append", "attend", "attend", "score"))
    if kind == "score":
        vocab = _log(rng, 500, 130000)
        return _score(_log(rng, 1, min(4096, 200_000_000 // vocab)), vocab, rng.choice((0, 1, 5, 20, 50)), rng.choice(("bf16", "bf16", "f16", "f32")))
    D = rng.choice((64, 128, 128, 96, 32))
    KV = rng.choice((1, 2, 4, 8, 12))
    H = KV * rng.choice((1, 2, 4, 5, 8))
    page, eight = rng.choice((16, 32, 64, 128, 256)), rng.random() < 0.7
    half, uneven = rng.choice(("bf16", "f16")), round(rng.random() * 0.9, 2)
    new = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 1500)))
    context = rng.choice((0, _log(rng, 16, 20000), _log(rng, 16, 20000)))
    if kind == "append":
        B = _log(rng, 1, max(1, min(64, 12000 * 1024 // ((new + context) * KV * D))))
        return _append(B, new, context, H, KV, D, page, rng.choice((0, D, D, D // 2)), half, eight, uneven)
    context = max(0, min(context, int(2e11 / (4 * H * D * new)) - new))                # not more than attend_pieces multiplies
    B = _log(rng, 1, max(1, min(64, 60_000_000 // ((new + context) * H * max(D, new)))))
    return _attend(B, new, context, H, KV, D, page, half, eight, uneven)


def _counts(c):
    """New tokens and keys (the new ones included) of each sequence: up to `uneven` of them are missing."""
    lengths, new = [], []
    for i in range(c["B"]):
        less = c["uneven"] * ((i + 0.25) * 0.6180339887 % 1.0)
        n = max(1, c["new"] - int(c["new"] * less))
        new.append(n)
        lengths.append(n + c["context"] - int(c["context"] * (c["uneven"] * ((i + 0.75) * 0.7548776662 % 1.0))))
    return lengths, new


def _quantised(x, scale):
    """x [..] as e4m3 at 2 ** (scale - 127)."""
    return torch.ldexp(x, 127 - scale.to(torch.int32)).to(E4M3)


def _exponent_of(amax):
    """The byte of the least scale of at least 2 ** -126 that holds amax within 448 = 1.75 * 2 ** 8."""
    m, e = torch.frexp(amax)                          # amax = m * 2 ** e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, e + 127, torch.ones_like(e)).clamp(1, 254).to(torch.uint8)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "score":
        x = torch.empty(c["rows"], c["vocab"], dtype=dt, device="cuda").normal_(0.0, 3.0, generator=g)
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        banned = torch.randint(0, c["vocab"], (8,), generator=g, device="cuda")       # tokens that the program does not allow
        x[:, banned[~torch.isin(banned, tokens)]] = float("-inf")
        return dict(case=c, logits=x, tokens=tokens)

    lengths, new = _counts(c)
    B, H, KV, D, page = c["B"], c["H"], c["KV"], c["D"], c["page"]
    T, width = sum(new), -(-max(lengths) // page)
    used = sum(-(-n // page) for n in lengths)
    pages = used + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:used].to(torch.int32)
    table, at = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(lengths):
        count = -(-n // page)
        table[b, :count] = order[at:at + count]
        at += count
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    # the layer's projection, of which q, k and v are views
    qkv = torch.empty(T, (H + 2 * KV) * D, dtype=dt, device="cuda").normal_(0.0, 1.0, generator=g)
    q, k, v = (t.view(T, -1, D) for t in qkv.split((H * D, KV * D, KV * D), dim=1))
    # what the cache holds already; where no token has been yet, whatever was in the memory
    held = dt if not c["eight"] else E4M3
    position = torch.arange(width * page, device="cuda")
    before = torch.tensor([n if c["kind"] == "attend" else n - m for n, m in zip(lengths, new)], device="cuda")
    filled = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    inside = (position[None] < before[:, None]).view(B, width, page)
    filled[table[table >= 0].long()] = inside[table >= 0]

    def cache():
        x = torch.empty(pages, KV, page, D, dtype=dt, device="cuda").normal_(0.0, 1.0, generator=g)
        x.mul_(torch.rand(pages, KV, 1, 1, generator=g, device="cuda").add_(0.5).to(dt))
        scale = None
        if c["eight"]:
            scale = _exponent_of((x * filled[:, None, :, None]).abs().amax((2, 3)).float())
            x = _quantised(x.float(), scale[..., None, None]).view(torch.uint8)
        x = torch.where(filled[:, None, :, None], x, torch.tensor(0x7F, dtype=torch.uint8, device="cuda") if c["eight"] else torch.tensor(float("nan"), dtype=dt, device="cuda"))
        return x.view(held), scale

    keys, key_scales = cache()
    values, value_scales = cache()
    values = values.view(torch.uint8 if c["eight"] else dt).view(pages, KV, page // 16, 16, D).transpose(3, 4).contiguous().view(held)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    state = dict(case=c, q=q, k=k, v=v, keys=keys, values=values, key_scales=key_scales, value_scales=value_scales, table=table, lengths=as_int(lengths),
                 starts=as_int(starts), most_new=max(new), most_keys=max(lengths), freqs=None)
    if c.get("rotated"):
        turn = torch.arange(c["rotated"] // 2, device="cuda", dtype=torch.float64) * (-2.0 / c["rotated"])
        angle = torch.arange(width * page, device="cuda", dtype=torch.float64)[:, None] * torch.pow(10000.0, turn)
        state["freqs"] = torch.cat((angle.cos(), angle.sin()), 1).float()
    return state


def _places(s):
    """Of every new token: its sequence, its position, the page and the slot that the position stands for."""
    starts, lengths, page = s["starts"].long(), s["lengths"].long(), s["case"]["page"]
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = (row[:, None] >= starts[None, 1:]).sum(1)
    p = lengths[b] - (starts[b + 1] - row)
    return b, p, s["table"].long()[b, p // page], p % page


def _rotated(x, cs):
    """x [T, heads, D] in fp32, the halves of its first R elements turned; cs [T, R]: cosines, sines."""
    h = cs.shape[1] // 2
    cos, sin = cs[:, None, :h], cs[:, None, h:]
    x1, x2 = x[..., :h], x[..., h:2 * h]
    return torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos, x[..., 2 * h:]), -1)


def _store(cache, scales, x, page, slot, by_token):
    """x [T, KV, D] into cache, with its values as `by_token` [pages, KV, page, D] lays them out; 8 bits: scales that may grow and values that follow them."""
    if scales is None:
        by_token[page, :, slot] = x.to(cache.dtype)
        return
    pages, KV, size, _ = by_token.shape
    first = torch.full((pages,), size, device="cuda").scatter_reduce_(0, page, slot, "amin")
    top = x.abs().amax(2)
    amax = torch.zeros(pages, KV, device="cuda").scatter_reduce_(0, page[:, None].expand(-1, KV), top, "amax")
    touched, fresh = (first < size)[:, None], (first == 0)[:, None]
    needed = _exponent_of(amax)
    grown = torch.where(touched, torch.where(fresh, needed, torch.maximum(needed, scales)), scales)
    old = (torch.arange(size, device="cuda") < first[:, None])[:, None, :, None] & (grown != scales)[:, :, None, None]
    raw = by_token.view(torch.uint8)
    moved = _quantised(by_token.float(), (127 + grown.int() - scales.int())[:, :, None, None]).view(torch.uint8)
    raw.copy_(torch.where(old, moved, raw))
    raw[page, :, slot] = _quantised(x, grown[page][:, :, None]).view(torch.uint8)
    scales.copy_(grown)


def _plain_append(s):
    _, p, page, slot = _places(s)
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["freqs"] is not None:
        cs = s["freqs"][p]
        q, k = _rotated(q, cs), _rotated(k, cs)
    keys, values = s["keys"], s["values"]
    _store(keys, s["key_scales"], k, page, slot, keys)
    kind = torch.uint8 if s["case"]["eight"] else values.dtype
    pages, KV, blocks, D, _ = values.shape
    by_token = values.view(kind).transpose(3, 4).contiguous().view(pages, KV, blocks * 16, D).view(values.dtype)
    _store(values, s["value_scales"], v, page, slot, by_token)
    values.view(kind).copy_(by_token.view(kind).view(pages, KV, blocks, 16, D).transpose(3, 4))
    return (q.to(s["q"].dtype) if s["freqs"] is not None else None), keys, values, s["key_scales"], s["value_scales"]


def _plain_attend(s):
    c = s["case"]
    T, H, D = s["q"].shape
    KV, page, B = c["KV"], c["page"], c["B"]
    G, L, N = H // KV, s["most_keys"], s["most_new"]
    b, p, _, _ = _places(s)
    place = b * N + (torch.arange(T, device="cuda") - s["starts"].long()[b])
    width = -(-L // page)
    pick = s["table"][:, :width].long().clamp(min=0)
    inside = torch.arange(width * page, device="cuda")[None] < s["lengths"][:, None]                        # [B, keys]

    def held(cache, scales):             # [B, KV, keys, D] in fp32, zero where no token is
        x = cache.float()
        if scales is not None:
            x = torch.ldexp(x, (scales.to(torch.int32) - 127)[:, :, None, None])
        x = x[pick].transpose(1, 2).reshape(B, KV, width * page, D)
        return torch.where(inside[:, None, :, None], x, 0.0)

    values = s["values"].view(torch.uint8 if c["eight"] else s["values"].dtype)
    k = held(s["keys"], s["key_scales"])
    v = held(values.transpose(3, 4).reshape(values.shape[0], KV, page, D).view(s["values"].dtype), s["value_scales"])
    q = torch.zeros(B * N, H, D, device="cuda").index_copy_(0, place, s["q"].float())
    q = q.view(B, N, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, D)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).view(B, KV, G, N, width * page)
    at = torch.zeros(B * N, dtype=torch.long, device="cuda").index_copy_(0, place, p).view(B, 1, 1, N, 1)
    x.masked_fill_(torch.arange(width * page, device="cuda") > at, float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    x.div_(x.sum(-1, keepdim=True))
    o = torch.matmul(x.view(B, KV, G * N, width * page), v).view(B, KV, G, N, D).permute(0, 3, 1, 2, 4).reshape(B * N, H, D)
    return o[place].to(s["q"].dtype)


def _plain_score(s):
    x = s["logits"].float()
    top = s["case"]["top"]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(1)
    log_total = total.log()
    log_p = d.gather(1, s["tokens"].long()[:, None])[:, 0] - log_total
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(1) / total
    if top == 0:
        return log_p, entropy
    value, index = torch.sort(d, dim=1, descending=True, stable=True)
    return log_p, entropy, value[:, :top] - log_total[:, None], index[:, :top].to(torch.int32)


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return _plain_append(s) if kind == "append" else _plain_attend(s) if kind == "attend" else _plain_score(s)
    from metalhlo_amd import kernels
    if kind == "score":
        return kernels.token_log_probs(s["logits"], s["tokens"], top=s["case"]["top"])
    cache = kernels.PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"])
    if kind == "attend":
        return kernels.paged_attention(s["q"], cache, s["table"], s["lengths"], s["starts"])
    if s["freqs"] is None:
        kernels.paged_append(cache, s["k"], s["v"], s["table"], s["lengths"], s["starts"])
        q = None
    else:
        q = kernels.paged_append(cache, s["k"], s["v"], s["table"], s["lengths"], s["starts"], q=s["q"], freqs=s["freqs"])
    return q, s["keys"], s["values"], s["key_scales"], s["value_scales"]


def work(case):
    c = case
    if c["kind"] == "score":
        n = c["rows"] * c["vocab"]
        return dict(bytes=SIZE[c["dtype"]] * n + c["rows"] * (12.0 + 8 * c["top"]), flops=6.0 * n)
    lengths, new = _counts(c)
    T, H, KV, D, e = sum(new), c["H"], c["KV"], c["D"], SIZE[c["dtype"]]
    held = 1 if c["eight"] else e
    if c["kind"] == "append":
        turned = 2.0 * e * T * H * D if c["rotated"] else 0.0
        return dict(bytes=turned + (e + held) * T * 2.0 * KV * D + 4.0 * T * c["rotated"], flops=3.0 * T * (H + KV) * c["rotated"] + 2.0 * T * KV * D)
    pairs = sum(m * (n - m) + m * (m + 1) / 2 for n, m in zip(lengths, new))
    return dict(bytes=2.0 * e * T * H * D + 2.0 * held * sum(lengths) * KV * D, flops=4.0 * pairs * H * D)


# ---- the definitions in 64 bits, sequence by sequence and head by head

def _e4m3(x):
    """The e4m3 number nearest to x, ties to even, in 64 bits (|x| <= 448)."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    c = s["case"]
    lengths, new = _counts(c)
    page, D, R = c["page"], c["D"], c["rotated"]
    q, keys = s["q"].double(), s["keys"].double()
    pages, KV = keys.shape[:2]
    values = s["values"].double().permute(0, 1, 2, 4, 3).reshape(pages, KV, page, D).clone()
    at = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        rows, pos = slice(at, at + m), torch.arange(n - m, n, device="cuda")
        at += m

        def turn(x):
            y = x.clone()
            if R:
                z = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous())
                f = s["freqs"][pos].double()
                z = z * torch.complex(f[:, :R // 2].contiguous(), f[:, R // 2:].contiguous())[:, None]
                y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
            return y
        q[rows] = turn(q[rows])
        for cache, scales, x in ((keys, s["key_scales"], turn(s["k"][rows].double())), (values, s["value_scales"], s["v"][rows].double())):
            first = n - m
            while first < n:
                last = min(n, (first // page + 1) * page)
                where, slot = int(s["table"][b, first // page]), first % page
                y = x[first - n + m:last - n + m].transpose(0, 1)
                if scales is not None:
                    big = y.abs().amax((1, 2))
                    e = torch.ceil(torch.log2(big / 448)).long().clamp(-126, 127)
                    e = torch.where(torch.ldexp(big.new_full((), 448.0), e) < big, e + 1, e)
                    was = scales[where].long() - 127
                    if slot:
                        e = torch.maximum(e, was)
                        cache[where][:, :slot] = _e4m3(torch.ldexp(cache[where][:, :slot], (was - e)[:, None, None]))
                    y = _e4m3(torch.ldexp(y, -e[:, None, None]))
                cache[where][:, slot:slot + last - first] = y
                first = last
    values = values.view(pages, KV, page // 16, 16, D).permute(0, 1, 2, 4, 3)
    return (q if R else None), keys, values, None, None


def _exact_attend(s):
    c = s["case"]
    lengths, new = _counts(c)
    KV, D, page = c["KV"], c["D"], c["page"]
    G, out, at = c["H"] // KV, torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        pages = s["table"][b, :-(-n // page)].long()
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(KV):
            k = s["keys"][pages, h].double().reshape(-1, D)[:n]
            v = s["values"][pages, h].double().transpose(2, 3).reshape(-1, D)[:n]
            if c["eight"]:
                k = k * torch.exp2(s["key_scales"][pages, h].double() - 127).repeat_interleave(page)[:n, None]
                v = v * torch.exp2(s["value_scales"][pages, h].double() - 127).repeat_interleave(page)[:n, None]
            for j in range(h * G, h * G + G):
                w = s["q"][at:at + m, j].double() @ k.t() / D ** 0.5
                out[at:at + m, j] = torch.softmax(w.masked_fill(hidden, float("-inf")), 1) @ v
        at += m
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    found = []
    for rows, tokens in zip(s["logits"].split(512), s["tokens"].long().split(512)):
        log_p = torch.log_softmax(rows.double(), 1)
        part = [log_p.gather(1, tokens[:, None])[:, 0], torch.special.entr(log_p.exp()).sum(1)]
        if case["top"]:
            part.append(torch.topk(log_p, case["top"], dim=1).values)
        found.append(part)
    got = [torch.cat(t) for t in zip(*found)]
    return (*got, None) if case["top"] else tuple(got)
