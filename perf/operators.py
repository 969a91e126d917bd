"""Serving operators as measured work: the 8-bit paged key/value cache (append, read back, attention over it) and the
verification of drafted tokens.

`run` computes them either in elementary torch operations in 32 bits (64 where a cumulative sum decides about a token), or, with
`own` set, by the calls a user of `whisper_amd` makes.  The cache is four tensors:

  k        int8 or float8_e4m3fn [pages, kv heads, P, D]      v  the same type [pages, kv heads, D, P] (transposed in its page)
  k_scale  float32 [pages, kv heads]                          v_scale  float32 [pages, kv heads]

a value is code * scale, a scale belongs to one page ("block") of P tokens and one head, and `table` [B, width] names the pages
of each sequence.  A code is x * r rounded once, r the scale's reciprocal as 32 bits hold it: the product has 48 bits, so it
is taken in 64, where nothing falls on the wrong side of a border."""
import torch

own = False

INT8, E4M3 = "int8", "e4m3"
FIT = {INT8: 127.5, E4M3: 448.0}      # a block keeps its scale while |x| <= FIT * scale: int8 rounds 127.5 down to 127
CODE = {INT8: torch.int8, E4M3: torch.float8_e4m3fn}
TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one window's newest token over the 1500 encoder frames of a 6-head decoder: latency is what counts
        {"name": "attend cross 1 window", "op": "attend", "B": 1, "H": 6, "Hkv": 6, "D": 64, "P": 64, "fmt": INT8, "dtype": "bf16",
         "T": 1, "ragged": False, "kv_lo": 1500, "kv": 1500, "causal": False},
        # the same for a full batch of 128 windows of a 12-head decoder: the stream that bounds decoding
        {"name": "attend cross 128 windows", "op": "attend", "B": 128, "H": 12, "Hkv": 12, "D": 64, "P": 64, "fmt": E4M3,
         "dtype": "bf16", "T": 1, "ragged": False, "kv_lo": 1500, "kv": 1500, "causal": False},
        # newest token over the text decoded so far, windows at every stage of their 448 positions, small pages, f32
        {"name": "attend self 32 windows f32", "op": "attend", "B": 32, "H": 8, "Hkv": 8, "D": 64, "P": 16, "fmt": INT8,
         "dtype": "f32", "T": 1, "ragged": False, "kv_lo": 1, "kv": 448, "causal": True},
        # four drafted tokens and the newest one, long contexts of unequal length, four query heads to a kv head
        {"name": "attend drafted long", "op": "attend", "B": 8, "H": 32, "Hkv": 8, "D": 128, "P": 64, "fmt": E4M3, "dtype": "bf16",
         "T": 5, "ragged": False, "kv_lo": 1000, "kv": 32768, "causal": True},
        # a 170-token prompt over the encoder frames in f32
        {"name": "attend prompt frames f32", "op": "attend", "B": 4, "H": 16, "Hkv": 16, "D": 64, "P": 64, "fmt": INT8,
         "dtype": "f32", "T": 170, "ragged": False, "kv_lo": 1500, "kv": 1500, "causal": False},
        # long causal prompts of unequal length behind a cached prefix
        {"name": "attend long prompts", "op": "attend", "B": 3, "H": 16, "Hkv": 4, "D": 64, "P": 128, "fmt": E4M3, "dtype": "bf16",
         "T": 4500, "ragged": True, "kv_lo": 4600, "kv": 5003, "causal": True},
        # the newest token of every window joins the cache
        {"name": "append token 128 windows", "op": "append", "B": 128, "Hkv": 12, "D": 64, "P": 64, "fmt": INT8, "dtype": "bf16",
         "T": 1, "ragged": False, "pos_lo": 169, "pos": 447},
        # the encoder frames of 32 windows are stored at once
        {"name": "append frames 32 windows", "op": "append", "B": 32, "Hkv": 12, "D": 64, "P": 64, "fmt": E4M3, "dtype": "bf16",
         "T": 1500, "ragged": False, "pos_lo": 0, "pos": 0},
        # prompts and drafted tokens of unequal length behind odd positions, f32
        {"name": "append ragged f32", "op": "append", "B": 16, "Hkv": 8, "D": 128, "P": 32, "fmt": INT8, "dtype": "f32",
         "T": 701, "ragged": True, "pos_lo": 3, "pos": 5001},
        # one window, four tokens from a drafter without probabilities
        {"name": "verify 1 window", "op": "verify", "B": 1, "N": 4, "V": 51864, "dtype": "f32", "kind": "logits", "draft": False,
         "temperature": 1.0, "ragged": False},
        # 64 windows, five tokens of a draft model, both models' logits
        {"name": "verify 64 windows", "op": "verify", "B": 64, "N": 5, "V": 51865, "dtype": "f32", "kind": "logits", "draft": True,
         "temperature": 0.8, "ragged": True},
        # greedy decoding: a drafted token stands while it is the arg-max
        {"name": "verify greedy 128 windows", "op": "verify", "B": 128, "N": 4, "V": 51866, "dtype": "bf16", "kind": "logits",
         "draft": False, "temperature": 0.0, "ragged": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))

    while True:
        op = rng.choice(("attend", "attend", "append", "verify"))
        if op == "verify":
            c = {"op": op, "B": spread(1, 128), "N": rng.randint(1, 8), "V": spread(1000, 140000), "dtype": rng.choice(("f32", "bf16")),
                 "kind": rng.choice(("logits", "logits", "probs")), "draft": rng.random() < 0.6,
                 "temperature": rng.choice((0.6, 0.8, 1.0, 1.3)), "ragged": rng.random() < 0.5}
            if c["kind"] == "probs":
                c["temperature"], c["dtype"] = 1.0, "f32"
            elif rng.random() < 0.2:
                c["temperature"], c["draft"] = 0.0, False
            if c["B"] * (2 * c["N"] + 1) * c["V"] > 64 * 11 * 51865:
                continue
            return c
        hkv = rng.choice((1, 2, 4, 6, 8, 12, 16, 20))
        c = {"op": op, "B": spread(1, 128), "Hkv": hkv, "D": rng.choice((64, 64, 128)), "P": rng.choice((16, 32, 64, 64, 128)),
             "fmt": rng.choice((INT8, E4M3)), "dtype": rng.choice(("bf16", "bf16", "f32")), "ragged": rng.random() < 0.4}
        if op == "append":
            c["T"] = rng.choice((1, spread(1, 8), spread(2, 1500)))
            c["pos"] = rng.choice((0, spread(1, 8000)))
            c["pos_lo"] = rng.randint(0, c["pos"])
            if c["B"] * c["T"] * hkv * c["D"] > 32 * 1500 * 12 * 64 or c["B"] * (c["T"] + c["pos"]) * hkv * c["D"] > 1 << 29:
                continue
            return c
        c["H"] = hkv * rng.choice((1, 1, 2, 4, 8))
        c["T"] = rng.choice((1, 1, spread(2, 8), spread(9, 1500)))
        c["kv"] = spread(1, 32768) if c["T"] == 1 else spread(c["T"], 32768)
        c["kv_lo"] = rng.randint(min(c["T"], c["kv"]), c["kv"])
        c["causal"] = rng.random() < 0.6
        flops = 4.0 * c["B"] * c["T"] * c["H"] * c["kv"] * c["D"]
        if c["B"] * c["kv"] * hkv * c["D"] > 128 * 1500 * 12 * 64 or flops > 1e11 or c["H"] > 64:
            continue
        return c


# ---- sizes that follow from a case alone ------------------------------------------------------------
def _lengths(n, lo, hi):
    """n lengths in [lo, hi], unequal, the first the largest."""
    return [hi] + [lo + int((hi - lo + 1) * ((i * 0.6180339887) % 1.0)) for i in range(1, n)]


def _plan(c):
    """Host-side lengths: tokens of each sequence in the call, and its length (attend) or position (append) before."""
    n = _lengths(c["B"], 1, c["T"]) if c["ragged"] else [c["T"]] * c["B"]
    if c["op"] == "append":
        return n, _lengths(c["B"], c["pos_lo"], c["pos"])
    return n, [max(a, b) if c["causal"] else a for a, b in zip(_lengths(c["B"], c["kv_lo"], c["kv"]), n)]


def work(c):
    es = {"bf16": 2, "f32": 4}[c["dtype"]]
    if c["op"] == "verify":
        rows = c["B"] * (c["N"] + 1 + (c["N"] if c["draft"] else 0))
        if c["kind"] == "probs":
            rows = c["B"] * (2 if c["draft"] else 1)
        return {"bytes": rows * c["V"] * es + 8 * c["B"] * (2 * c["N"] + 2), "flops": 4.0 * rows * c["V"]}
    n, at = _plan(c)
    if c["op"] == "append":
        new = sum(n) * c["Hkv"] * c["D"] * 2
        back = sum(p + m - p // c["P"] * c["P"] for p, m in zip(at, n)) * c["Hkv"] * c["D"] * 2
        return {"bytes": new * (es + 1) + back * (es + 1), "flops": 4.0 * (new + back)}
    cached = sum(at) * c["Hkv"] * (c["D"] * 2 + 8.0 / c["P"])
    pairs = sum(m * L - (m * (m - 1) // 2 if c["causal"] else 0) for m, L in zip(n, at)) * c["H"]
    return {"bytes": cached + sum(n) * c["H"] * (c["D"] * es * 2 + 4), "flops": 4.0 * pairs * c["D"]}


# ---- inputs -----------------------------------------------------------------------------------------
def _quantise(x, fmt):
    """x [..., P, D] f32 -> codes, scale [...] as a block stored at once has them."""
    amax = x.abs().amax((-1, -2))
    s = _base(amax, fmt)
    return _coded(x, s, fmt), s


def _values(gen, dev, *shape):
    """Keys or values: normal, a few channels several times larger than the rest, as projections have them."""
    x = torch.randn(shape, generator=gen, device=dev)
    return x * (1.0 + 5.0 * (torch.rand(shape[-1], generator=gen, device=dev) < 0.06))


def _cache(c, gen, dev, width):
    """A cache whose pages hold tokens throughout (also behind the sequences' ends), in a shuffled order, some pages unused."""
    B, Hkv, D, P = c["B"], c["Hkv"], c["D"], c["P"]
    pages = B * width + 3
    k, ks = _quantise(_values(gen, dev, pages, Hkv, P, D), c["fmt"])
    v, vs = _quantise(_values(gen, dev, pages, Hkv, P, D), c["fmt"])
    table = torch.randperm(pages, generator=gen, device=dev)[: B * width].view(B, width).to(torch.int32)
    v = v.view(torch.uint8).transpose(2, 3).contiguous().view(CODE[c["fmt"]])
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table}


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _starts(n):
    out = [0]
    for m in n:
        out.append(out[-1] + m)
    return out


def prepare(c, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 7919 + 17)
    dt = TYPE[c["dtype"]]
    st = {"case": c}
    if c["op"] == "verify":
        B, N, V = c["B"], c["N"], c["V"]
        # next-token scores of a trained decoder: a few likely tokens, a long tail; the drafter's are a perturbed copy
        x = torch.randn(B, N + 1, V, generator=gen, device=dev) * 2.5
        x += 9.0 * (torch.rand(B, N + 1, V, generator=gen, device=dev) < 4.0 / V)
        y = x[:, :N] + 0.7 * torch.randn(B, N, V, generator=gen, device=dev)
        x, y = x.to(dt), y.to(dt)
        noise = torch.rand(B, N, V, generator=gen, device=dev)
        t = c["temperature"] or 0.1
        drafted = (y.float() / t - torch.log(-torch.log(noise.clamp(1e-20, 1 - 1e-7)))).argmax(-1)
        st["drafted"] = drafted.to(torch.int32)
        if c["kind"] == "probs":
            x, y = torch.softmax(x.float(), -1).to(dt), torch.softmax(y.float(), -1).to(dt)
        st["target"], st["draft"] = x, y if c["draft"] else None
        st["uniforms"] = torch.rand(B, N + 1, generator=gen, device=dev)
        st["n_drafted"] = _i32(_lengths(B, 0, N), dev) if c["ragged"] else None
        return st
    n, at = _plan(c)
    P = c["P"]
    last = [p + m for p, m in zip(at, n)] if c["op"] == "append" else at
    width = max((m + P - 1) // P for m in last) + 1
    st.update(_cache(c, gen, dev, width))
    st["tok_start"] = _i32(_starts(n), dev) if c["ragged"] else None
    N = sum(n)
    row_b = torch.repeat_interleave(torch.arange(c["B"], device=dev), torch.tensor(n, device=dev), output_size=N)
    st["row_b"] = row_b
    st["row_t"] = torch.arange(N, device=dev) - torch.tensor(_starts(n)[:-1], device=dev)[row_b]
    st["n_of"], st["at"] = torch.tensor(n, device=dev), _i32(at, dev)
    lead = (N,) if c["ragged"] else (c["B"], c["T"])
    if c["op"] == "attend":
        st["q"] = torch.randn(*lead, c["H"], c["D"], generator=gen, device=dev).to(dt)
        return st
    st["new_k"] = _values(gen, dev, *lead, c["Hkv"], c["D"]).to(dt)
    st["new_v"] = _values(gen, dev, *lead, c["Hkv"], c["D"]).to(dt)
    # the blocks the call touches, and the tokens that are read back: all of those blocks up to the sequences' new ends
    touched = [(b, j) for b in range(c["B"]) for j in range(at[b] // P, (at[b] + n[b] - 1) // P + 1)]
    st["blk_b"] = torch.tensor([b for b, _ in touched], device=dev)
    st["blk_j"] = torch.tensor([j for _, j in touched], device=dev)
    first = [p // P * P for p in at]
    back = [p + m - f for p, m, f in zip(at, n, first)]
    st["back_first"], st["back_start"], st["back_n"] = _i32(first, dev), _i32(_starts(back), dev), sum(back)
    bb = torch.repeat_interleave(torch.arange(c["B"], device=dev), torch.tensor(back, device=dev), output_size=sum(back))
    st["back_b"] = bb
    st["back_pos"] = torch.arange(sum(back), device=dev) - torch.tensor(_starts(back)[:-1], device=dev)[bb] + st["back_first"][bb]
    return st


# ---- plain forms --------------------------------------------------------------------------------------
def _two_to(e):
    """2^e in float32, exactly (a power function need not be exact)."""
    return ((e.clamp(-126, 127).int() + 127) << 23).view(torch.float32)


def _base(amax, fmt):
    """The scale of a block that begins with values up to amax."""
    if fmt == INT8:
        s = (amax / 127.0).clamp(min=2.0 ** -126)
    else:
        m, e = torch.frexp(amax.double() / 448.0)
        s = _two_to(e - (m == 0.5).to(e.dtype))
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _to_code(y, fmt):
    if fmt == INT8:
        return torch.round(y).clamp(-127, 127).to(torch.int8)
    return y.clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)      # powers of two as scales: nothing is lost before


def _coded(x, s, fmt):
    """Codes of x [..., a, b] under the scales s [...]."""
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    return _to_code(x.double() * r.double()[..., None, None], fmt)


def _pages(x, pages):
    """x[pages] for code tensors of any type."""
    return x.view(torch.uint8)[pages].view(x.dtype).float()


def _store(codes, scale, x, st, transposed):
    """Appends x to one of the cache's halves; x [N, Hkv, D] f32."""
    c = st["case"]
    P, fmt = c["P"], c["fmt"]
    b, j = st["blk_b"], st["blk_j"]
    page = st["table"].long()[b, j]
    pos = st["at"].long()[b, None]
    p = j[:, None] * P + torch.arange(P, device=x.device)                       # [blocks, P] positions
    is_new = (p >= pos) & (p < pos + st["n_of"][b, None])
    is_old = p < pos
    start = torch.cumsum(st["n_of"], 0) - st["n_of"]
    row = (start[b, None] + p - pos).clamp(0, x.shape[0] - 1)
    xn = x[row].permute(0, 2, 1, 3) * is_new[:, None, :, None]                   # [blocks, Hkv, P, D]
    old = _pages(codes, page)
    old = old.transpose(2, 3) if transposed else old
    s = scale[page]
    amax = xn.abs().amax((-1, -2))
    fresh = (j * P >= st["at"].long()[b])[:, None] | (s == 0)
    need = amax.double() / (FIT[fmt] * torch.where(fresh, torch.ones_like(s), s).double())
    m, e = torch.frexp(need)
    up = torch.where(~fresh & (need > 1), e - (m == 0.5).to(e.dtype), torch.zeros_like(e))
    s = torch.where(fresh, _base(amax, fmt), s * _two_to(up))
    kept = torch.where(up[..., None, None] > 0, _to_code(old * _two_to(-up)[..., None, None], fmt).float(), old)
    fill = _coded(xn, s, fmt).float()
    new = torch.where(is_new[:, None, :, None], fill, torch.where(is_old[:, None, :, None], kept, old))
    new = (new.transpose(2, 3) if transposed else new).contiguous().to(codes.dtype)
    codes.view(torch.uint8)[page] = new.view(torch.uint8)
    scale[page] = s


def _token_values(codes, scale, st, transposed, dt):
    """The values of the tokens that are read back, [tokens, Hkv, D]."""
    P = st["case"]["P"]
    b, p = st["back_b"], st["back_pos"].long()
    page = st["table"].long()[b, p // P]
    u = codes.view(torch.uint8)
    x = u[page, :, :, p % P] if transposed else u[page, :, p % P]
    return (x.contiguous().view(codes.dtype).float() * scale[page][:, :, None]).to(dt)


def _attend(st):
    c = st["case"]
    B, H, Hkv, D, P = c["B"], c["H"], c["Hkv"], c["D"], c["P"]
    dev, dt = st["q"].device, st["q"].dtype
    q = st["q"].reshape(-1, H, D).float()
    table = st["table"].long()
    k = (_pages(st["k"], table) * st["k_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    v = (_pages(st["v"], table) * st["v_scale"][table][..., None, None]).transpose(3, 4).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    S, kv = k.shape[2], st["at"].long()
    j = torch.arange(S, device=dev)
    v = torch.where((j < kv[:, None])[:, None, :, None], v, torch.zeros((), device=dev))
    T = c["T"]
    qp = torch.zeros(B, T, H, D, device=dev)
    qp[st["row_b"], st["row_t"]] = q
    qp = qp.view(B, T, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * (H // Hkv), D)
    s = torch.matmul(qp, k.transpose(2, 3)) * D ** -0.5                          # [B, Hkv, T * G, S]
    seen = kv[:, None].expand(B, T)
    if c["causal"]:
        seen = kv[:, None] - st["n_of"][:, None] + 1 + torch.arange(T, device=dev)
    hide = j >= seen[:, None, :, None, None]                                     # [B, 1, T, 1, S]
    s = s.view(B, Hkv, T, H // Hkv, S).masked_fill_(hide, float("-inf")).view(B, Hkv, -1, S)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp_(s.sub_(m))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = m + torch.log(total)
    o = o.view(B, Hkv, T, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)[st["row_b"], st["row_t"]]
    lse = lse.view(B, Hkv, T, H // Hkv).permute(0, 2, 1, 3).reshape(B, T, H)[st["row_b"], st["row_t"]]
    return {"out": o.to(dt).view(st["q"].shape), "lse": lse.view(st["q"].shape[:-1])}


def _verify(st):
    c = st["case"]
    B, N, V, x, d = c["B"], c["N"], c["V"], st["target"], st["drafted"].long()
    dev = x.device
    n = st["n_drafted"].long() if st["n_drafted"] is not None else torch.full((B,), N, device=dev)
    at = torch.arange(N, device=dev)
    all_b = torch.arange(B, device=dev)
    if c["temperature"] == 0:
        x = x.float()
        ids = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)
        ok = (ids[:, :N] == d) & (at < n[:, None])
        acc = ok.int().cumprod(1).sum(1)
        nxt = ids[all_b, acc]
    else:
        def rows(y):
            y = y.double()
            if c["kind"] == "probs":
                return y
            y = torch.exp((y - y.amax(-1, keepdim=True)) / c["temperature"])
            return y / y.sum(-1, keepdim=True)

        p, u = rows(x), st["uniforms"].double()
        q = rows(st["draft"]) if st["draft"] is not None else None
        pd = p[:, :N].gather(2, d[..., None])[..., 0]
        qd = q.gather(2, d[..., None])[..., 0] if q is not None else torch.ones_like(pd)
        ok = (u[:, :N] * qd < pd) & (at < n[:, None])
        acc = ok.int().cumprod(1).sum(1)
        i = acc.clamp(max=N - 1)
        pr = p[all_b, acc]
        qr = q[all_b, i] if q is not None else (torch.arange(V, device=dev) == d[all_b, i][:, None]).double()
        w = torch.where((acc < n)[:, None], (pr - qr).clamp(min=0), pr)
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, pr)
        cum = w.cumsum(-1)
        nxt = (cum <= u[:, N:] * cum[:, -1:]).sum(-1)
        last = torch.where(w > 0, torch.arange(V, device=dev), -1).amax(-1)
        nxt = torch.minimum(nxt, last)
    out = torch.where(at < acc[:, None], d, -1)
    out = torch.cat([out, torch.full((B, 1), -1, device=dev)], 1)
    out[all_b, acc] = nxt
    return {"accepted": acc.to(torch.int32), "tokens": out.to(torch.int32)}


def run(st):
    c = st["case"]
    if own:
        if c["op"] == "verify":
            from whisper_amd import speculative
            acc, tokens = speculative.verify_draft(st["target"], st["drafted"], st["uniforms"], draft=st["draft"],
                                                   n_drafted=st["n_drafted"], temperature=c["temperature"], probs=c["kind"] == "probs")
            return {"accepted": acc, "tokens": tokens}
        from whisper_amd import kv8
        cache = kv8.KV8Cache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        if c["op"] == "attend":
            out, lse = kv8.attention(st["q"], cache, st["table"], st["at"], tok_start=st["tok_start"], causal=c["causal"],
                                     return_lse=True)
            return {"out": out, "lse": lse}
        kv8.append(cache, st["new_k"], st["new_v"], st["table"], st["at"], tok_start=st["tok_start"])
        k, v = kv8.read(cache, st["table"], st["back_first"], st["back_n"], tok_start=st["back_start"], dtype=TYPE[c["dtype"]])
        return {"k": k, "v": v}
    if c["op"] == "verify":
        return _verify(st)
    if c["op"] == "attend":
        return _attend(st)
    tokens = (-1, c["Hkv"], c["D"])
    _store(st["k"], st["k_scale"], st["new_k"].reshape(tokens).float(), st, False)
    _store(st["v"], st["v_scale"], st["new_v"].reshape(tokens).float(), st, True)
    dt = TYPE[c["dtype"]]
    return {"k": _token_values(st["k"], st["k_scale"], st, False, dt), "v": _token_values(st["v"], st["v_scale"], st, True, dt)}


# ---- the definitions in 64 bits, sequence by sequence ---------------------------------------------------
def _exact_half(codes, scale, x, st, transposed):
    """Appends in 64 bits, block by block of positions: the codes are those of the definition (a scale and its reciprocal are held in 32 bits)."""
    c = st["case"]
    P, fmt, n, at = c["P"], c["fmt"], *_plan(c)
    table, starts, out = st["table"].tolist(), _starts(n), []
    x = x.reshape(-1, c["Hkv"], c["D"]).double()
    power = lambda e: (2.0 ** e).float().double()  # noqa: E731  (rounding to 32 bits makes the power exact)
    for b in range(c["B"]):
        first = at[b] // P
        pages = table[b][first: (at[b] + n[b] - 1) // P + 1]
        old = codes.view(torch.uint8)[pages].view(codes.dtype).double()
        old = old.transpose(2, 3) if transposed else old
        nb, before = len(pages), at[b] - first * P
        old = old.transpose(1, 2).reshape(nb * P, c["Hkv"], c["D"])
        full = torch.zeros_like(old)
        full[before: before + n[b]] = x[starts[b]: starts[b] + n[b]]
        top = full.abs().view(nb, P, c["Hkv"], c["D"]).amax((1, 3))
        sc = scale[pages].double()
        if fmt == INT8:
            begin = (top / 127).clamp(min=2.0 ** -126).float().double()
        else:
            begin = power(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448) - 1e-12).clamp(min=-126))
        begin = torch.where(top > 0, begin, torch.zeros_like(begin))
        k = torch.ceil(torch.log2((top / (FIT[fmt] * sc.clamp(min=1e-300))).clamp(min=1e-300)) - 1e-12).clamp(min=0)
        k = torch.where((sc == 0) | ((torch.arange(nb, device=x.device) > 0) | (before == 0))[:, None], torch.zeros_like(k), k)
        begins = (torch.arange(nb, device=x.device) > 0)[:, None] | (before == 0) | (sc == 0)
        sc = torch.where(begins, begin, sc * power(k))
        each = lambda t: t.repeat_interleave(P, 0)[:, :, None]  # noqa: E731
        at_new = torch.arange(nb * P, device=x.device)
        is_new = ((at_new >= before) & (at_new < before + n[b]))[:, None, None]
        r = torch.where(sc > 0, 1 / sc, torch.zeros_like(sc)).float().double()
        y = torch.where(is_new, full * each(r), old * power(-each(k)))
        if fmt == INT8:
            y = torch.round(y).clamp(-127, 127)
        else:
            step = power(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4.0)
            y = (torch.round(y / step) * step).clamp(-448, 448)
        out.append((y * each(sc))[: before + n[b]])
    return torch.cat(out)


def exact(c, seed):
    if c["op"] == "verify":
        return None                                      # whole numbers
    st = prepare(c, seed)
    if c["op"] == "append":
        return {"k": _exact_half(st["k"], st["k_scale"], st["new_k"], st, False),
                "v": _exact_half(st["v"], st["v_scale"], st["new_v"], st, True)}
    n, kv = _plan(c)
    starts, G = _starts(n), c["H"] // c["Hkv"]
    q = st["q"].reshape(-1, c["H"], c["D"]).double()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for b in range(c["B"]):
        pages = st["table"][b, : -(-kv[b] // c["P"])].long()
        for g in range(c["Hkv"]):
            k = st["k"].view(torch.uint8)[pages, g].view(st["k"].dtype).double() * st["k_scale"][pages, g].double()[:, None, None]
            v = st["v"].view(torch.uint8)[pages, g].view(st["v"].dtype).double() * st["v_scale"][pages, g].double()[:, None, None]
            k, v = k.reshape(-1, c["D"])[: kv[b]], v.transpose(1, 2).reshape(-1, c["D"])[: kv[b]]
            for h in range(g * G, g * G + G):
                for t0 in range(0, n[b], 1024):
                    t = torch.arange(t0, min(n[b], t0 + 1024), device=q.device)
                    s = q[starts[b] + t, h] @ k.T / c["D"] ** 0.5
                    if c["causal"]:
                        s = s.masked_fill(torch.arange(kv[b], device=q.device) > kv[b] - n[b] + t[:, None], float("-inf"))
                    lse[starts[b] + t, h] = torch.logsumexp(s, -1)
                    out[starts[b] + t, h] = torch.softmax(s, -1) @ v
    return {"out": out.view(st["q"].shape), "lse": lse.view(st["q"].shape[:-1])}
