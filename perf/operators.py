"""The KV cache held in 4 bits, as a serving program uses it: rows written (`append`), values read back (`read`), and
attention over the cache for single tokens, for a few rows per sequence and for prompt chunks (`attention`).

The arena is `[pages][kv_heads][18 head_dim]` bytes, 16 tokens a page.  A page of one head holds K codes (8 head_dim bytes),
V codes (8 head_dim), K scales and V scales (binary16, one for 32 dimensions of a token).  With G = 32-dimension group,
groups in blocks of four (`sub`, `w`; two where a head has only two), token j = 8 c + 2 t + e of the page:
  K codes   [sub][j][t'][w][4 bytes]       nibble i of the word is dimension 32 G + 8 t' + i
  V codes   [sub][c][g][t][w][e][2 bytes]  nibble i of the half word is dimension 32 G + 8 i + g
  K scales  [j][G]
  V scales  [c][t][G][e]
A value is scale x (code - 8).  A row's group is quantised by its value x of largest magnitude (the first of them): scale =
x / -8 in binary16 with 7 significant bits, code = floor(value / scale + 1/2) + 8 in 0..15.
"""
import math

import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence's new row of one layer, written and taken back: the smallest call, latency alone
        dict(name="write-1", kind="write", rows=1, kv_heads=8, head_dim=128, dtype="f32", pages=64, spread=False),
        # a prompt chunk's rows of one layer as the prompt's own attention would see them
        dict(name="write-2048", kind="write", rows=2048, kv_heads=8, head_dim=128, dtype="bf16", pages=4096, spread=False),
        # an odd prompt with heads of 64, its pages anywhere
        dict(name="write-777-hd64", kind="write", rows=777, kv_heads=4, head_dim=64, dtype="f16", pages=512, spread=True),
        # a finished context handed to an executor with an F16 cache
        dict(name="read-16384", kind="read", rows=16384, kv_heads=8, head_dim=128, dtype="f16", pages=2048),
        # a very long one in the type of this package's host operators, not whole pages
        dict(name="read-60001", kind="read", rows=60001, kv_heads=8, head_dim=128, dtype="f32", pages=8192),
        # a decode step of the 0.6B model: one sequence, its new row and the attention of it
        dict(name="step-1x1024", kind="step", seqs=1, rows=1, keys=1024, ragged=False, q_heads=16, kv_heads=8, head_dim=128,
             dtype="bf16", window=0, pad=0),
        # a decode step of the 8B model with sixty-four ragged sequences and three padding rows, in this package's F32
        dict(name="step-64x1500", kind="step", seqs=64, rows=1, keys=1500, ragged=True, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f32", window=0, pad=3),
        # long contexts in a batch: what the 4-bit cache is for
        dict(name="step-16x32768", kind="step", seqs=16, rows=1, keys=32768, ragged=True, q_heads=32, kv_heads=8, head_dim=128,
             dtype="bf16", window=0, pad=0),
        # one sequence of 65,536 keys: the long axis has to be split
        dict(name="step-1x65536", kind="step", seqs=1, rows=1, keys=65536, ragged=False, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", window=0, pad=0),
        # four proposed tokens per sequence checked at once, 32B heads, a sliding window
        dict(name="step-40x4-window", kind="step", seqs=40, rows=4, keys=9000, ragged=True, q_heads=64, kv_heads=8, head_dim=128,
             dtype="f16", window=4096, pad=0),
        # an odd prompt of the 0.6B model from nothing, in this package's F32
        dict(name="chunk-777", kind="step", seqs=1, rows=777, keys=777, ragged=False, q_heads=16, kv_heads=8, head_dim=128,
             dtype="f32", window=0, pad=0),
        # a prompt chunk of the 8B model behind 14,336 tokens: the largest
        dict(name="chunk-2048-behind-14336", kind="step", seqs=1, rows=2048, keys=16384, ragged=False, q_heads=32, kv_heads=8,
             head_dim=128, dtype="bf16", window=0, pad=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    kind = rng.choice(["write", "read", "decode", "decode", "few", "chunk", "chunk"])
    if kind in ("write", "read"):
        rows = _log(rng, 1, 8192) if kind == "write" else _log(rng, 100, 60000)
        return dict(kind=kind, rows=rows, kv_heads=rng.choice([1, 2, 4, 8, 8]), head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype,
                    pages=rows // PAGE + rng.randint(2, 500), **(dict(spread=rng.random() < 0.5) if kind == "write" else {}))
    q_heads, kv_heads = rng.choice([(16, 8), (32, 8), (32, 8), (64, 8), (8, 1), (12, 4), (5, 5), (16, 1)])
    window = rng.choice([0, 0, 0, _log(rng, 100, 5000)])
    if kind == "chunk":
        # a chunk alone or behind a prefix, one to three sequences
        seqs = rng.choice([1, 1, 2, 3])
        rows = _log(rng, 33, 2048 // seqs)
        keys = rows + rng.choice([0, _log(rng, 16, 14000 // seqs)])
        return dict(kind="step", seqs=seqs, rows=rows, keys=keys, ragged=seqs > 1, q_heads=min(q_heads, 32), kv_heads=kv_heads,
                    head_dim=rng.choice([64, 128, 128]), dtype=dtype, window=window, pad=rng.choice([0, 5]))
    keys = _log(rng, 16, 65536)
    seqs = max(1, min(96, _log(rng, 1, max(2, 500000 // keys))))
    rows = 1 if kind == "decode" else rng.randint(2, 8)
    return dict(kind="step", seqs=seqs, rows=rows, keys=keys, ragged=rng.random() < 0.7, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=rng.choice([64, 128, 128, 128, 256]), dtype=dtype, window=window, pad=rng.choice([0, 0, 7]))


# ---- inputs ------------------------------------------------------------------------------------------------------
def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _codes(gen, pages, kv_heads, head_dim):
    """Codes 0..15 [pages][kv_heads][16][head_dim] as quantised rows have them: bell shaped, every group with an extreme one."""
    x = torch.randn((pages, kv_heads, PAGE, head_dim), generator=gen, device=DEVICE, dtype=torch.float16)
    x = x.mul_(2.9).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    x[..., ::32] = 0
    return x


def _scales(gen, pages, kv_heads, head_dim):
    """Scales [pages][kv_heads][16][groups], binary16 with 7 significant bits, of either sign."""
    x = torch.randn((pages, kv_heads, PAGE, head_dim // 32), generator=gen, device=DEVICE)
    s = (0.3 * torch.exp(0.3 * x)).to(torch.float16).view(torch.int16)
    s = ((s + 8) & ~15).view(torch.float16)
    return torch.where(x.sin() > 0, s, -s)


def _blocks(head_dim):
    words = min(4, head_dim // 32)
    return head_dim // 32 // words, words


def _pack(k_codes, k_scales, v_codes, v_scales):
    p, h, _, d = k_codes.shape
    sub, w = _blocks(d)
    k = k_codes.view(p, h, PAGE, sub, w, 4, 4, 2)
    k = (k[..., 0] | (k[..., 1] << 4)).permute(0, 1, 3, 2, 5, 4, 6)                  # [sub][j][t'][w][byte]
    v = v_codes.view(p, h, 2, 4, 2, sub, w, 2, 2, 8)                                 # c t e sub w byte nibble g
    v = (v[:, :, :, :, :, :, :, :, 0] | (v[:, :, :, :, :, :, :, :, 1] << 4)).permute(0, 1, 5, 2, 8, 3, 6, 4, 7)   # [sub][c][g][t][w][e][byte]
    vs = v_scales.view(p, h, 2, 4, 2, d // 32).permute(0, 1, 2, 3, 5, 4)
    parts = [k.reshape(p, h, 8 * d), v.reshape(p, h, 8 * d), k_scales.reshape(p, h, -1).view(torch.uint8),
             vs.reshape(p, h, -1).view(torch.uint8)]
    return torch.cat(parts, dim=2)


def _arena(gen, pages, kv_heads, head_dim, keep=None):
    """The cache's bytes; with a dict in `keep` the codes and scales behind them too."""
    made = [f(gen, pages, kv_heads, head_dim) for f in (_codes, _scales, _codes, _scales)]
    if keep is not None:
        keep.update(zip(("k_codes", "k_scales", "v_codes", "v_scales"), made))
    return _pack(*made)


def _lengths(case):
    """Keys of each sequence, its new rows among them."""
    n, keys, rows = case["seqs"], case["keys"], case["rows"]
    if not case["ragged"]:
        return [keys] * n
    # from the longest down to a third of it, in an order that is not sorted; one sequence in eleven has only its new rows
    out = [max(rows, keys - (i * 7919 % n) * (2 * keys // 3) // n) for i in range(n)]
    return [rows if i % 11 == 5 else x for i, x in enumerate(out)]


def _inputs(case, seed, keep=None):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, h, d = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    if case["kind"] in ("write", "read"):
        n = case["rows"]
        order = torch.randperm(case["pages"], generator=gen, device=DEVICE)
        at = torch.arange(n, device=DEVICE)
        if case.get("spread"):
            slots = torch.randperm(case["pages"] * PAGE, generator=gen, device=DEVICE)[:n]     # a row anywhere
        else:
            at = at + 5 if n + 5 <= case["pages"] * PAGE else at                                # not from a page's first row on
            slots = order[at // PAGE] * PAGE + at % PAGE
        s = dict(case=case, slots=slots.to(torch.int32), cache=_arena(gen, case["pages"], h, d, keep))
        if case["kind"] == "write":
            channel = torch.exp(0.4 * torch.randn((h, d), generator=gen, device=DEVICE))
            s["k"] = (torch.randn((n, h, d), generator=gen, device=DEVICE) * channel).to(dtype)
            s["v"] = _randn(gen, (n, h, d), dtype, 0.7)
        return s
    n, rows, pad = case["seqs"], case["rows"], case["pad"]
    lengths = _lengths(case)
    per_sequence = max(-(-x // PAGE) for x in lengths) + 1
    pages = sum(-(-x // PAGE) for x in lengths) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    tables = torch.zeros((n, per_sequence), dtype=torch.int32, device=DEVICE)
    first = 0
    for i, x in enumerate(lengths):
        count = -(-x // PAGE)
        tables[i, :count] = order[first:first + count]
        first += count
    total = n * rows + pad
    at = torch.tensor(lengths, device=DEVICE).view(n, 1) - rows + torch.arange(rows, device=DEVICE)        # positions [n][rows]
    slots = torch.gather(tables.long(), 1, at // PAGE) * PAGE + at % PAGE
    slots = torch.cat([slots.view(-1), torch.full((pad,), -1, device=DEVICE)])                              # padding rows are not written
    return dict(case=case, tables=tables, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
                cu_rows=torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device=DEVICE), slots=slots.to(torch.int32),
                cache=_arena(gen, pages, h, d, keep), k=_randn(gen, (total, h, d), dtype), v=_randn(gen, (total, h, d), dtype, 0.7),
                q=_randn(gen, (total, case["q_heads"], d), dtype, 2.0), out=torch.full((total, case["q_heads"], d), 0.25, dtype=dtype, device=DEVICE))


def prepare(case, seed):
    return _inputs(case, seed)


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from ribn_b200 import kvq4
    case, cache = s["case"], s["cache"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "read":
        return kvq4.read(cache, s["slots"], dtype=dtype)
    kvq4.append(cache, s["k"], s["v"], s["slots"])
    if case["kind"] == "write":
        return kvq4.read(cache, s["slots"], dtype=dtype)
    return kvq4.attention(cache, s["q"], s["tables"], s["lengths"], s["cu_rows"], max_rows=case["rows"], max_keys=case["keys"],
                          window=case["window"], out=s["out"])


def _run_plain(s):
    case, cache = s["case"], s["cache"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "read":
        return _plain_read(cache, s["slots"], dtype)
    _plain_append(cache, s["k"], s["v"], s["slots"])
    if case["kind"] == "write":
        return _plain_read(cache, s["slots"], dtype)
    return _plain_attention(cache, s["q"], s["tables"], s["lengths"], s["cu_rows"], case["rows"], case["window"], s["out"])


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _sections(cache):
    d = cache.shape[2] // 18
    return d, cache[..., :8 * d], cache[..., 8 * d:16 * d], cache[..., 16 * d:17 * d], cache[..., 17 * d:]


def _unpack(cache):
    """K and V of pages [..][kv_heads][18 d] as F32 values [..][kv_heads][16][d]."""
    lead, d = cache.shape[:-1], cache.shape[-1] // 18
    sub, w = _blocks(d)
    flat = cache.reshape(-1, 1, 18 * d)
    n = flat.shape[0]
    _, kc, vc, ks, vs = _sections(flat)
    kc = kc.reshape(n, sub, PAGE, 4, w, 4)
    k = torch.stack([kc & 15, kc >> 4], dim=-1).permute(0, 2, 1, 4, 3, 5, 6).reshape(n, PAGE, d // 32, 32)
    vc = vc.reshape(n, sub, 2, 8, 4, w, 2, 2)
    v = torch.stack([vc & 15, vc >> 4], dim=-1).permute(0, 2, 4, 6, 1, 5, 7, 8, 3).reshape(n, PAGE, d // 32, 32)
    ks = ks.reshape(n, d).contiguous().view(torch.float16).view(n, PAGE, d // 32, 1).float()
    vs = vs.reshape(n, d).contiguous().view(torch.float16).view(n, 2, 4, d // 32, 2).permute(0, 1, 2, 4, 3).reshape(n, PAGE, d // 32, 1).float()
    k, v = ((k.float() - 8) * ks).view(*lead, PAGE, d), ((v.float() - 8) * vs).view(*lead, PAGE, d)
    return k, v


def _quantise(x):
    """Codes 0..15 and scales of rows [n][h][d].  The quotients are formed in 64 bits, so that none lands on the wrong side of a border."""
    n, h, d = x.shape
    g = x.float().view(n, h, d // 32, 32)
    size = g.abs()
    first = (size == size.amax(dim=3, keepdim=True)) * torch.arange(32, 0, -1, device=x.device)      # the first of the largest
    top = g.gather(3, first.argmax(dim=3, keepdim=True))
    bits = (top / -8).to(torch.float16).view(torch.int16).int()
    bits = (bits & 0x8000) | torch.clamp(((bits & 0x7fff) + 8) & ~15, max=0x6300)
    scale = torch.where(bits >= 0x8000, bits - 0x10000, bits).to(torch.int16).view(torch.float16)
    q = torch.floor(g.double() / torch.where(scale == 0, torch.ones_like(scale), scale).double() + 0.5).clamp(-8, 7)
    q = torch.where(scale == 0, torch.zeros_like(q), q)
    return (q + 8).to(torch.uint8).view(n, h, d), scale.squeeze(3)


def _plain_append(cache, k, v, slots):
    d = k.shape[2]
    sub, w = _blocks(d)
    keep = slots >= 0
    k, v, at = k[keep], v[keep], slots[keep].long()
    n, h = k.shape[:2]
    page, j = at // PAGE, at % PAGE
    c, t, e = j // 8, j % 8 // 2, j % 2
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    kc = kc.view(n, h, sub, w, 4, 4, 2)
    kc = (kc[..., 0] | (kc[..., 1] << 4)).permute(0, 1, 2, 4, 3, 5).reshape(n, h, sub, 16 * w)      # [sub][t'][w][byte]
    vc = vc.view(n, h, sub, w, 2, 2, 8)
    vc = (vc[:, :, :, :, :, 0] | (vc[:, :, :, :, :, 1] << 4)).permute(0, 1, 2, 5, 3, 4)             # [sub][g][w][byte]
    _, to_k, to_v, to_ks, to_vs = _sections(cache)
    to_k.unflatten(2, (sub, PAGE, 16 * w))[page, :, :, j] = kc
    to_v.unflatten(2, (sub, 2, 8, 4, w, 2, 2))[page, :, :, c, :, t, :, e] = vc
    to_ks.unflatten(2, (PAGE, d // 16))[page, :, j] = ks.contiguous().view(torch.uint8).view(n, h, d // 16)
    to_vs.unflatten(2, (2, 4, d // 32, 2, 2))[page, :, c, t, :, e] = vs.contiguous().view(torch.uint8).view(n, h, d // 32, 2)


def _plain_read(cache, slots, dtype):
    at = slots.long().clamp(min=0)
    k, v = _unpack(cache[at // PAGE])
    pick = (at % PAGE).view(-1, 1, 1, 1).expand(-1, k.shape[1], 1, k.shape[3])
    live = (slots >= 0).view(-1, 1, 1)
    return tuple((x.gather(2, pick).squeeze(2) * live).to(dtype) for x in (k, v))


def _plain_attention(cache, q, tables, lengths, cu_rows, max_rows, window, out):
    n, d = lengths.shape[0], q.shape[2]
    k, v = _unpack(cache[tables.long()])                                                            # [n][pages][h][16][d]
    h = k.shape[2]
    k, v = (x.transpose(1, 2).reshape(n, h, -1, d) for x in (k, v))
    at = cu_rows[:-1].long().view(n, 1) + torch.arange(max_rows, device=q.device)
    live = at < cu_rows[1:].long().view(n, 1)
    rows = q[torch.where(live, at, 0)].float().view(n, max_rows, h, -1, d)
    group = rows.shape[3]
    rows = rows.permute(0, 2, 1, 3, 4).reshape(n, h, max_rows * group, d) * (1 / math.sqrt(d))
    pos = lengths.view(n, 1) - (cu_rows[1:] - cu_rows[:-1]).view(n, 1) + torch.arange(max_rows, device=q.device)
    key = torch.arange(k.shape[2], device=q.device)
    see = key <= pos.unsqueeze(2)
    if window > 0:
        see = see & (key > pos.unsqueeze(2) - window)
    score = torch.matmul(rows, k.transpose(2, 3)).view(n, h, max_rows, group, -1)
    score.masked_fill_(~see.view(n, 1, max_rows, 1, -1), -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = score.sum(dim=-1, keepdim=True)
    result = torch.matmul(score.view(n, h, max_rows * group, -1), v).view(n, h, max_rows, group, d)
    result = result / torch.where(total > 0, total, torch.ones_like(total))
    result = result.permute(0, 2, 1, 3, 4).reshape(n, max_rows, h * group, d)
    out[at[live]] = result[live].to(out.dtype)
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    size, h, d = (4 if case["dtype"] == "f32" else 2), case["kv_heads"], case["head_dim"]
    row = 2 * h * d                                   # values of K and V of a token
    if case["kind"] in ("write", "read"):
        n = case["rows"]
        moved = n * row * size + n * row * 9 // 16    # values out, or back; the cache's side of it
        return dict(bytes=moved * (2 if case["kind"] == "write" else 1), flops=0)
    rows, window = case["rows"], case["window"]
    seen = read = 0
    for keys in _lengths(case):
        first = keys - rows                           # rows see first + 1 .. keys, or the window of those
        if window:
            seen += sum(min(window, first + 1 + i) for i in range(rows))
        else:
            seen += rows * first + rows * (rows + 1) // 2
        read += min(keys, window + rows - 1) if window else keys
    total = case["seqs"] * rows
    moved = read * row * 9 // 16 + total * row * size + total * row * 9 // 16 + 2 * total * case["q_heads"] * d * size
    return dict(bytes=moved, flops=4 * seen * case["q_heads"] * d)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _to_values(codes, scales):
    """[pages][h][16][d] codes and their scales as 64-bit values [pages * 16][h][d]."""
    x = (codes.double() - 8.0).unflatten(3, (-1, 32)) * scales.double().unsqueeze(4)
    return x.flatten(3).transpose(1, 2).flatten(0, 1)


def _rounded_row(x):
    """The cached values of rows [n][h][d]: by the definition, 64 bits throughout."""
    g = x.double().unflatten(2, (-1, 32))
    size = g.abs()
    most = size.max(dim=3, keepdim=True).values
    places = torch.arange(32, device=x.device).expand_as(g)
    place = torch.where(size == most, places, 32).min(dim=3, keepdim=True).values
    wanted = (torch.gather(g, 3, place) / -8.0).half().double()       # the binary16 next to it ..
    # .. and of that the nearest with 7 significant bits, half away from zero (steps of 2^-20 below the normal range), up to 896
    exponent = torch.floor(torch.log2(wanted.abs().clamp(min=2.0 ** -14)))
    step = torch.exp2(exponent - 6)
    scale = wanted.sign() * (torch.floor(wanted.abs() / step + 0.5) * step).clamp(max=896.0)
    code = torch.floor(g / torch.where(scale == 0, torch.ones_like(scale), scale) + 0.5).clamp(-8, 7)
    return (code * scale).flatten(2)


def exact(case, seed):
    made = {}
    s = _inputs(case, seed, made)
    if case["kind"] == "write":
        keep = (s["slots"] >= 0).view(-1, 1, 1)
        return tuple(_rounded_row(x) * keep for x in (s["k"], s["v"]))
    if case["kind"] == "read":
        at = s["slots"].long()
        out = []
        for name in ("k", "v"):
            codes, scales = made[name + "_codes"], made[name + "_scales"]
            x = (codes[at // PAGE, :, at % PAGE].double() - 8.0).unflatten(2, (-1, 32)) * scales[at // PAGE, :, at % PAGE].double().unsqueeze(3)
            out.append(x.flatten(2))
        return tuple(out)
    new = {name: _rounded_row(s[name]) for name in ("k", "v")}
    q, out = s["q"].double(), s["out"].double()
    group, rows, window = case["q_heads"] // case["kv_heads"], case["rows"], case["window"]
    for i, keys in enumerate(_lengths(case)):
        pages = s["tables"][i, :-(-keys // PAGE)].long()
        own_rows = slice(i * rows, (i + 1) * rows)
        cached = []
        for name in ("k", "v"):
            x = _to_values(made[name + "_codes"][pages], made[name + "_scales"][pages])[:keys]
            cached.append(torch.cat([x[:keys - rows], new[name][own_rows]]))
        for j in range(case["kv_heads"]):
            heads = slice(j * group, (j + 1) * group)
            score = torch.einsum("rgd,td->rgt", q[own_rows, heads], cached[0][:, j]) / math.sqrt(case["head_dim"])
            place = torch.arange(keys, device=q.device).view(1, 1, keys)
            last = (keys - rows + torch.arange(rows, device=q.device)).view(rows, 1, 1)
            hidden = place > last
            if window:
                hidden = hidden | (place <= last - window)
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), dim=2)
            out[own_rows, heads] = torch.einsum("rgt,td->rgd", weight, cached[1][:, j])
    return out
