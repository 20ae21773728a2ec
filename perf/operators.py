"""A key/value cache held in 4 bits and the attention that reads it: cases, their plain form, and the answer in 64 bits.

Four operators, as a serving program calls them:

* "write": the step's [q; k; v] rows rotated, q stored, k and v quantised into the pages of their requests; what was stored
  is then read back (what is held in 4 bits is compared as the values that it stands for);
* "read": rows of the cache read back as plain rows of the compute dtype;
* "decode": attention of single tokens, each over its own request's positions;
* "prompt": attention of prompt portions, causal, over what the cache holds of their requests.

The cache.  32 dims of a head of one position share a scale s and a zero z: with lo = min(0, smallest), hi = max(0, largest),
s is (hi - lo) / 15 rounded up to a half-precision number of six significant bits (at most 2112), z = rint(-lo / s) and
n = rint(x / s) + z, both kept in 0 .. 15; the number held is s (n - z).  Keys lie [page][kv head][slot][dims / 2 bytes] with
[slot][dims / 32] scales behind them, values [page][kv head][slot / 8][dims] words of eight positions with
[slot / 8][dims / 32][8] scales behind them.  A word of eight numbers e0 .. e7 is the sum of e(2i) << 4i and
e(2i+1) << (16 + 4i), rotated left by 6; a scale's 16 bits are the half-precision number's, with z in the low four.
"""
import math

import torch

own = False

if_own = {}          # dtype -> the framework's kernels, loaded where `own` is true

GROUP = 32           # dims that share a scale
LARGEST = 2112.0     # the largest scale


# ---------------------------------------------------------------------------- cases


def _case(name, op, dtype, heads, kv_heads, dim, page, spans, window=0, pad=0):
    """`spans`: a text, one "tokens@start" a request (a decoded token at position p: "1@p"); `pad`: tokens at no position behind them."""
    case = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, spans=spans, window=window, pad=pad)
    return dict(case, name=name) if name else case


def _spans(case):
    return [tuple(int(n) for n in part.split("@")) for part in case["spans"].split()]


def _text(spans):
    return " ".join(f"{n}@{start}" for n, start in spans)


def listed():
    return [
        # a decoding step of eight requests of the 7B sizes: a layer's write, where latency counts
        _case("write: 8 single tokens", "write", "bfloat16", 28, 4, 128, 16, _text((1, 2048 + 17 * i) for i in range(8))),
        # a prompt of 8,192 tokens in one step
        _case("write: a prompt of 8192", "write", "bfloat16", 28, 4, 128, 16, "8192@0"),
        # portions of several requests of uneven lengths, true 32-bit rows, small heads
        _case("write: ragged portions, float32", "write", "float32", 14, 2, 64, 64, "777@0 1@4001 130@63 1001@515 5@7"),
        # one request's rows taken out of the cache (to look at what the 4 bits kept)
        _case("read: one request of 301", "read", "bfloat16", 28, 4, 128, 16, "301@0"),
        # eight long requests taken out
        _case("read: 8 requests of 16384", "read", "bfloat16", 28, 4, 128, 64, _text([(16384, 0)] * 8)),
        # one user: the latency of a decoded token's attention
        _case("decode: 1 token at 2100", "decode", "bfloat16", 28, 4, 128, 16, "1@2100"),
        # the benchmark's long-context batch
        _case("decode: 8 tokens at 32768", "decode", "bfloat16", 28, 4, 128, 16, _text((1, 32768 + i) for i in range(8))),
        # a busy server: 64 requests of 64 to 4,000 positions, 14B heads, two rows of padding
        _case("decode: 64 ragged tokens", "decode", "bfloat16", 40, 8, 128, 64,
              _text((1, 64 + (i * 2477) % 3937) for i in range(64)), pad=2),
        # a window and small heads, true 32-bit rows
        _case("decode: 16 tokens in a window, float32", "decode", "float32", 14, 2, 64, 32,
              _text((1, 333 + 701 * i) for i in range(16)), window=4096),
        # short prompts of a chat side by side with portions far into their requests
        _case("prompt: ragged portions", "prompt", "bfloat16", 28, 4, 128, 16, "512@1536 37@0 300@4099 129@64 2@900"),
        # a long prompt in one step
        _case("prompt: 8192 tokens", "prompt", "bfloat16", 28, 4, 128, 16, "8192@0"),
        # small heads in a window, true 32-bit rows
        _case("prompt: 1000 tokens in a window, float32", "prompt", "float32", 14, 2, 64, 64, "1000@0 333@1001", window=700),
    ]


HEADS = [(28, 4), (40, 8), (14, 2), (16, 2), (8, 8), (12, 1), (7, 1), (40, 2)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    heads, kv_heads = rng.choice(HEADS)
    dim, page = rng.choice([64, 128, 128]), rng.choice([8, 16, 32, 64, 128])
    window = _log(rng, 16, 8192) if op in ("decode", "prompt") and rng.random() < 0.3 else 0
    pad = rng.choice([0, 0, 1, 3])
    if op == "decode":
        n = _log(rng, 1, 96)
        longest = min(33000, 262144 * 4 // (n * kv_heads))
        spans = [(1, _log(rng, 1, longest) - 1) for _ in range(n)]
    elif op == "prompt":
        n = _log(rng, 1, 6)
        budget = 8192 * 8192 // 2 * 28 // n
        spans = []
        for _ in range(n):
            tokens = _log(rng, 2, int(8192 * min(1.0, (28 / heads) ** 0.5)) // n)
            spans.append((tokens, min(_log(rng, 1, 16000) - 1, max(0, budget // (heads * tokens) - tokens))))
    else:
        n = _log(rng, 1, 8)
        spans = [(_log(rng, 1, (8192 if op == "write" else 131072 * 4 // kv_heads // 2) // n), _log(rng, 1, 9000) - 1) for _ in range(n)]
        pad = pad if op == "write" else 0
    return _case("", op, dtype, heads, kv_heads, dim, page, _text(spans), window, pad)


def _seen(case, pos):
    return pos + 1 if case["window"] == 0 else min(pos + 1, case["window"])


def work(case):
    spans, nh, nkv, hd = _spans(case), case["heads"], case["kv_heads"], case["dim"]
    elem = 2 if case["dtype"] == "bfloat16" else 4
    tokens = sum(n for n, _ in spans)
    rows = tokens + case["pad"]
    row = nkv * 2 * (hd // 2 + hd // 16)            # a position's keys and values
    if case["op"] == "write":
        # the rows in, the rotation's table, q out, the 4-bit rows out, and these read back as plain rows
        moved = rows * ((nh + 2 * nkv) * hd * elem + hd * 4 + nh * hd * elem) + tokens * (2 * row + 2 * nkv * hd * elem)
        return dict(bytes=moved, flops=rows * (3 * (nh + nkv) * hd + 10 * nkv * hd))
    if case["op"] == "read":
        return dict(bytes=tokens * (row + 2 * nkv * hd * elem), flops=tokens * 4 * nkv * hd)
    pairs = sum(_seen(case, start + i) for n, start in spans for i in range(n))
    positions = sum(min(start + n, _seen(case, start) + n - 1) for n, start in spans)
    return dict(bytes=positions * row + rows * 2 * nh * hd * elem, flops=4 * nh * hd * pairs)


# ---------------------------------------------------------------------------- inputs


def _pack(numbers):
    """int32 words of eight numbers each, from whole numbers [..., 8]."""
    n = numbers.to(torch.int64)
    word = torch.zeros(n.shape[:-1], dtype=torch.int64, device=n.device)
    for i in range(4):
        word |= (n[..., 2 * i] << (4 * i)) | (n[..., 2 * i + 1] << (16 + 4 * i))
    word = ((word << 6) | (word >> 26)) & 0xFFFFFFFF
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _unpack(words):
    """Whole numbers [..., 8] from int32 words."""
    w = words.to(torch.int64) & 0xFFFFFFFF
    w = ((w >> 6) | (w << 26)) & 0xFFFFFFFF
    return torch.stack([(w >> (4 * (i // 2) + 16 * (i % 2))) & 15 for i in range(8)], dim=-1)


def _quantise(x):
    """Float32 rows [..., dims] -> (numbers [..., dims], scale words [..., dims / 32])."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    finite = torch.isfinite(g).all(-1)
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    want = (hi - lo) / torch.full_like(lo, 15.0)            # (a tensor: by a number it would be a product with 1 / 15)
    half = want.clamp(max=LARGEST).to(torch.float16)
    bits = half.view(torch.int16).to(torch.int32)
    bits = torch.where(half.float() < want.clamp(max=LARGEST), bits + 1, bits)      # the half-precision number above, where it was rounded down
    bits = (bits + 31) & ~31                                                        # up to six significant bits
    s = bits.to(torch.int16).view(torch.float16).float()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / safe).clamp(0, 15)
    n = (torch.round(g / safe[..., None]) + z[..., None]).clamp(0, 15)
    n = torch.where(finite[..., None], n, torch.zeros_like(n)).to(torch.int32)
    word = torch.where(finite, bits | z.nan_to_num().to(torch.int32), torch.full_like(bits, 0x7FE0))
    return n.reshape(x.shape), word


def _values(numbers, words):
    """What numbers [..., dims] with scale words [..., dims / 32] stand for, float32."""
    s = (words & 0x7FE0).to(torch.int16).view(torch.float16).float()
    z = (words & 15).float()
    g = numbers.reshape(*numbers.shape[:-1], -1, GROUP).float()
    return (s[..., None] * (g - z[..., None])).reshape(numbers.shape)


def _row_bytes(dim):
    return dim // 2 + dim // 16


def _as_bytes(t):
    return t.contiguous().view(torch.uint8).flatten(1)


def _key_pages(rows, page):
    """Pages of keys [pages, heads, page, row bytes] from rows [pages, heads, page, dims]."""
    pages, heads, _, dim = rows.shape
    n, words = _quantise(rows)
    packed = _as_bytes(_pack(n.reshape(pages * heads, page * dim // 8, 8)))
    scales = _as_bytes(words.to(torch.int16).reshape(pages * heads, -1))
    return torch.cat([packed, scales], dim=1).view(pages, heads, page, _row_bytes(dim))


def _value_pages(rows, page):
    pages, heads, _, dim = rows.shape
    n, words = _quantise(rows)
    octets = n.reshape(pages * heads, page // 8, 8, dim).transpose(2, 3)
    packed = _as_bytes(_pack(octets).reshape(pages * heads, -1))
    scales = _as_bytes(words.to(torch.int16).reshape(pages * heads, page // 8, 8, dim // GROUP).transpose(2, 3).reshape(pages * heads, -1))
    return torch.cat([packed, scales], dim=1).view(pages, heads, page, _row_bytes(dim))


def _split(cache, dim, keys):
    """A cache's words and scale words, as [pages, heads, page, ...] of positions (numbers [.., dims], words [.., dims / 32])."""
    pages, heads, page, row = cache.shape
    flat = cache.reshape(pages * heads, page * row)
    cut = page * dim // 2
    words = flat[:, :cut].contiguous().view(torch.int32)
    scales = flat[:, cut:].contiguous().view(torch.int16).to(torch.int32) & 0xFFFF
    if keys:
        n = _unpack(words).reshape(pages, heads, page, dim)
        return n, scales.reshape(pages, heads, page, dim // GROUP)
    n = _unpack(words).reshape(pages * heads, page // 8, dim, 8).transpose(2, 3).reshape(pages, heads, page, dim)
    return n, scales.reshape(pages * heads, page // 8, dim // GROUP, 8).transpose(2, 3).reshape(pages, heads, page, dim // GROUP)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    spans, nh, nkv, hd, page = _spans(case), case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = getattr(torch, case["dtype"])
    positions, rows = [], []
    for r, (n, start) in enumerate(spans):
        positions += range(start, start + n)
        rows += [r] * n
    positions += [-1] * case["pad"]
    rows += [0] * case["pad"]
    T = len(positions)
    longest = max(start + n for n, start in spans)
    width = -(-longest // page)
    held = [-(-(start + n) // page) for n, start in spans]
    order = torch.randperm(sum(held) + 3, generator=torch.Generator().manual_seed(seed))
    table, at = torch.zeros((len(spans), width), dtype=torch.int32), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n].to(torch.int32)
        at += n
    n_pages = len(order)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    state = dict(case=case, positions=i32(positions), seq_rows=i32(rows), block_table=table.to(dev), spans=spans)
    # channels of keys differ widely in size, as a model's do, and their means are not zero
    size = torch.exp(0.7 * torch.randn((nkv, hd), generator=g, device=dev))
    mean = 0.5 * torch.randn((nkv, hd), generator=g, device=dev) * size
    scale = hd ** -0.5
    if case["op"] == "write":
        qkv = torch.randn((T, nh + 2 * nkv, hd), generator=g, device=dev)
        qkv[:, nh:nh + nkv] = qkv[:, nh:nh + nkv] * size + mean
        state["qkv"] = qkv.reshape(T, -1).to(dtype)
        freqs = 1000000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=dev) / hd)
        angle = state["positions"].double()[:, None] * freqs
        state["table"] = torch.stack([angle.sin(), angle.cos()], dim=-1).float()
        state["keys"] = torch.full((n_pages, nkv, page, _row_bytes(hd)), 255, dtype=torch.uint8, device=dev)
        state["values"] = torch.full_like(state["keys"], 255)
    else:
        keys = torch.empty((n_pages, nkv, page, _row_bytes(hd)), dtype=torch.uint8, device=dev)
        values = torch.empty_like(keys)
        part = max(1, 2 ** 24 // (nkv * page * hd))
        for a in range(0, n_pages, part):
            n = min(part, n_pages - a)
            x = torch.randn((n, nkv, page, hd), generator=g, device=dev)
            keys[a:a + n] = _key_pages(x * size[:, None] + mean[:, None], page)
            values[a:a + n] = _value_pages(torch.randn((n, nkv, page, hd), generator=g, device=dev), page)
        state["keys"], state["values"] = keys, values
        if case["op"] != "read":
            state["q"] = torch.randn((T, nh * hd), generator=g, device=dev).to(dtype)
            state["scale"] = scale
    if own:
        if case["dtype"] not in if_own:
            from axon_amd.kernels import kernels
            if_own[case["dtype"]] = kernels(case["dtype"])
        k = state["k"] = if_own[case["dtype"]]
        if case["op"] == "decode":
            state["work"] = i32(k.kv4_decode_work(positions, case["window"]))
            state["chunks"] = k.kv4_decode_chunks(positions, case["window"])
            state["partial"] = torch.empty(k.kv4_decode_workspace(T, nh, hd, state["chunks"]), dtype=torch.float32, device=dev)
        elif case["op"] == "prompt":
            firsts = [sum(n for n, _ in spans[:r]) for r in range(len(spans))]
            tiles = k.kv4_prefill_tiles([(f, n, start) for f, (n, start) in zip(firsts, spans)], case["window"], nh, nkv)
            state["tiles"] = i32(tiles)
            state["partial"] = torch.empty(k.kv4_prefill_workspace(tiles, nh, hd), dtype=torch.float32, device=dev)
    return state


# ---------------------------------------------------------------------------- one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    c, k = state["case"], state["k"]
    nh, nkv, hd, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    pos, rows, table, keys, values = (state[n] for n in ("positions", "seq_rows", "block_table", "keys", "values"))
    dtype, T = getattr(torch, c["dtype"]), pos.numel()
    if c["op"] in ("write", "read"):
        out = []
        if c["op"] == "write":
            q = torch.empty((T, nh * hd), dtype=dtype, device="cuda")
            k.rope_kv4_write(state["qkv"], q, state["table"], pos, rows, table, keys, values, nh, nkv, hd, hd, page)
            out = [q]
        n = T - c["pad"]
        k_rows, v_rows = (torch.empty((n, nkv, hd), dtype=dtype, device="cuda") for _ in range(2))
        k.kv4_read(keys, values, table, pos[:n], rows[:n], k_rows, v_rows, nkv, hd, page)
        return out + [k_rows, v_rows]
    out = torch.empty((T, nh * hd), dtype=dtype, device="cuda")
    common = (state["q"], nh * hd, keys, values, table, pos, rows, out)
    sizes = (nh, nkv, hd, page, c["window"], state["scale"])
    if c["op"] == "decode":
        return k.kv4_attention_decode(*common, T, state["partial"], state["chunks"], *sizes, work=state["work"])
    if c["pad"]:
        out[T - c["pad"]:].zero_()            # rows of no tile are left as they are
    return k.kv4_attention_prefill(*common, state["tiles"], state["partial"], *sizes)


def _slots(state, at):
    """(page, slot) of the tokens `at`."""
    page = state["case"]["page"]
    pos, rows = state["positions"][at].long(), state["seq_rows"][at].long()
    return state["block_table"][rows, pos // page].long(), pos % page


def _run_plain(state):
    c = state["case"]
    nh, nkv, hd, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dtype, T = getattr(torch, c["dtype"]), state["positions"].numel()
    if c["op"] in ("write", "read"):
        return _plain_rows(state, nh, nkv, hd, page, dtype, T)
    out = torch.zeros((T, nh * hd), dtype=dtype, device="cuda")
    first = 0
    for r, (n, start) in enumerate(state["spans"]):
        end = start + n
        low = max(0, start + 1 - c["window"]) // page if c["window"] else 0
        pages = state["block_table"][r, low:-(-end // page)].long()
        k, v = (_values(*_split(state[name][pages], hd, name == "keys")).transpose(0, 1).reshape(nkv, -1, hd) for name in ("keys", "values"))
        base, k, v = low * page, k[:, :end - low * page], v[:, :end - low * page]
        at = torch.arange(base, end, device="cuda")
        q = state["q"][first:first + n].float().view(n, nkv, nh // nkv, hd)
        part = max(1, 2 ** 26 // ((nh // nkv) * (end - base)))
        for h in range(nkv):
            turned = k[h].t().contiguous()
            for a in range(0, n, part):
                b = min(n, a + part)
                s = torch.matmul(q[a:b, h].reshape(-1, hd), turned).view(b - a, nh // nkv, -1) * state["scale"]
                pos = torch.arange(start + a, start + b, device="cuda")[:, None]
                hidden = at > pos
                if c["window"]:
                    hidden = hidden | (at <= pos - c["window"])
                s = s.masked_fill(hidden[:, None], -math.inf)
                e = torch.exp(s - s.amax(-1, keepdim=True))
                o = torch.matmul(e.reshape(-1, end - base), v[h]).view(b - a, nh // nkv, hd) / e.sum(-1, keepdim=True)
                out.view(T, nkv, nh // nkv, hd)[first + a:first + b, h] = o.to(dtype)
        first += n
    return out


def _plain_rows(state, nh, nkv, hd, page, dtype, T):
    out, n = [], T - state["case"]["pad"]
    where = _slots(state, slice(0, n))
    if state["case"]["op"] == "write":
        rows = state["qkv"].float().view(T, nh + 2 * nkv, hd)
        sin, cos = state["table"][..., 0][:, None], state["table"][..., 1][:, None]
        a, b = rows[:, :nh + nkv, :hd // 2], rows[:, :nh + nkv, hd // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        out = [turned[:, :nh].reshape(T, -1).to(dtype)]
        for name, x in (("keys", turned[:n, nh:]), ("values", rows[:n, nh + nkv:])):
            numbers, words = _quantise(x)
            _store(state, name, numbers, words, where, hd, page)
    # read back what lies in the tokens' slots
    for name in ("keys", "values"):
        pages, inverse = torch.unique(where[0], return_inverse=True)
        parts, step = [], max(1, 2 ** 24 // (nkv * page * hd))
        for a in range(0, len(pages), step):
            parts.append(_values(*_split(state[name][pages[a:a + step]], hd, name == "keys")))
        held = torch.cat(parts)
        out.append(held[inverse, :, where[1]].to(dtype))
    return out


def _store(state, name, numbers, words, where, hd, page):
    cache = state[name]
    pages, nkv, _, row = cache.shape
    flat = cache.view(pages, nkv, page * row)
    cut = page * hd // 2
    used, inverse = torch.unique(where[0], return_inverse=True)
    n_all, w_all = _split(cache[used], hd, name == "keys")
    n_all, w_all = n_all.contiguous(), w_all.contiguous()
    n_all[inverse, :, where[1]] = numbers.long()
    w_all[inverse, :, where[1]] = words
    if name == "keys":
        packed, scales = _pack(n_all.reshape(len(used), nkv, -1, 8)), w_all
    else:
        packed = _pack(n_all.reshape(len(used), nkv, page // 8, 8, hd).transpose(3, 4))
        scales = w_all.reshape(len(used), nkv, page // 8, 8, hd // GROUP).transpose(3, 4)
    flat[used, :, :cut] = packed.reshape(len(used) * nkv, -1).contiguous().view(torch.uint8).view(len(used), nkv, cut)
    scales = torch.where(scales >= 2 ** 15, scales - 2 ** 16, scales).to(torch.int16)
    flat[used, :, cut:] = scales.reshape(len(used) * nkv, -1).contiguous().view(torch.uint8).view(len(used), nkv, -1)


# ---------------------------------------------------------------------------- the answer in 64 bits


def _exact_held(cache, dim, keys, pages, slots):
    """Numbers held at (page, slot), float64 [n, heads, dims], nibble by nibble out of the bytes."""
    heads, page = cache.shape[1], cache.shape[2]
    flat = cache.view(cache.shape[0], heads, -1)
    d = torch.arange(dim, device=cache.device)
    s, word_at, inside = slots[:, None], None, None
    if keys:
        word_at, inside = s * (dim // 8) + d // 8, (d % 8).expand(len(slots), dim)
        meta_at = page * dim // 2 + 2 * (s * (dim // 32) + d // 32)
    else:
        word_at, inside = (s // 8) * dim + d, (s % 8).expand(len(slots), dim)
        meta_at = page * dim // 2 + 2 * (((s // 8) * (dim // 32) + d // 32) * 8 + s % 8)
    place = (inside // 2 * 4 + inside % 2 * 16 + 6) % 32          # where the number's lowest bit lies in its word
    out = torch.zeros((len(slots), heads, dim), dtype=torch.float64, device=cache.device)
    for h in range(heads):
        of = flat[:, h]
        number = torch.zeros_like(place)
        for bit in range(4):
            b = (place + bit) % 32
            byte = of[pages[:, None], word_at * 4 + b // 8].long()
            number += ((byte >> (b % 8)) & 1) << bit
        meta = of[pages[:, None], meta_at].long() | (of[pages[:, None], meta_at + 1].long() << 8)
        exponent, fraction = (meta >> 10) & 31, (meta & 0x3E0).double() / 1024.0
        scale = torch.where(exponent > 0, (1.0 + fraction) * torch.exp2((exponent - 15).double()), fraction * 2.0 ** -14)
        scale = torch.where(exponent == 31, torch.full_like(scale, math.nan), scale)
        out[:, h] = scale * (number - (meta & 15)).double()
    return out


def _exact_quantised(x):
    """What rows [..., dims] become, float64."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = torch.minimum(g.min(-1).values, torch.zeros((), device=x.device)), torch.maximum(g.max(-1).values, torch.zeros((), device=x.device))
    want = torch.clamp((hi - lo) / 15, max=LARGEST)
    _, e = torch.frexp(want)                                       # want = m 2^e, m in [0.5, 1): six bits are steps of 2^(e - 6)
    step = torch.exp2(torch.clamp(e - 6, min=-19).double())
    s = torch.ceil(want / step) * step
    unit = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.clamp(torch.round(-lo / unit), 0, 15)[..., None]
    n = torch.clamp(torch.round(g / unit[..., None]) + z, 0, 15)
    return (s[..., None] * (n - z)).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    nh, nkv, hd, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    T, spans = state["positions"].numel(), state["spans"]
    n = T - case["pad"]
    if case["op"] == "write":
        x = state["qkv"].double().view(T, -1, hd)
        sin, cos = state["table"].double().unbind(-1)
        turned = x[:, :nh + nkv].clone()
        for i in range(hd // 2):
            a, b = x[:, :nh + nkv, i], x[:, :nh + nkv, i + hd // 2]
            turned[:, :, i] = a * cos[:, i:i + 1] - b * sin[:, i:i + 1]
            turned[:, :, i + hd // 2] = a * sin[:, i:i + 1] + b * cos[:, i:i + 1]
        return [turned[:, :nh].reshape(T, -1), _exact_quantised(turned[:n, nh:]), _exact_quantised(x[:n, nh + nkv:])]
    if case["op"] == "read":
        pages = torch.stack([state["block_table"][r, p // page] for r, p in zip(*(t.tolist() for t in (state["seq_rows"], state["positions"])))]) \
            if n < 4096 else state["block_table"].flatten()[state["seq_rows"].long() * state["block_table"].shape[1] + state["positions"].long() // page]
        slots = state["positions"].long() % page
        return [torch.cat([_exact_held(state[name], hd, name == "keys", pages[a:a + 65536].long(), slots[a:a + 65536])
                           for a in range(0, n, 65536)]) for name in ("keys", "values")]
    out, first = torch.zeros((T, nh, hd), dtype=torch.float64, device="cuda"), 0
    for r, (count, start) in enumerate(spans):
        p = torch.arange(start + count, device="cuda")
        pages = state["block_table"][r].long()[p // page]
        k, v = (_exact_held(state[name], hd, name == "keys", pages, p % page) for name in ("keys", "values"))
        q = state["q"][first:first + count].double().view(count, nh, hd)
        part = max(1, 2 ** 27 // len(p))
        for h in range(nh):
            kv = h // (nh // nkv)
            for a in range(0, count, part):
                mine = torch.arange(start + a, start + min(count, a + part), device="cuda")[:, None]
                seen = (p <= mine) & ((p > mine - case["window"]) if case["window"] else (p >= 0))
                s = q[a:a + part, h] @ k[:, kv].t() * state["scale"]
                out[first + a:first + min(count, a + part), h] = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), dim=-1) @ v[:, kv]
        first += count
    return out.view(T, nh * hd)
