"""Cases that measure the low-precision serving operators, with their plain forms.

Four operators of one decoding step, each in two forms:

  norm     residual addition, RMS norm, and an output in 8 bits with scales
  cache    writing keys and values into a paged cache in 4 bits, and reading
           them back
  attend   attention of new queries over that cache
  product  activations times 4-bit weights with group scales

`own` chooses the form of run(): false computes the operator with elementary
torch operations in 32 bits, true makes the calls of the b200k package.  Both
forms read the same bytes: the layouts of the cache and of the weights are
written down here once in torch (cache_bytes, weight_tiles).
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "ouroboros-kernelsmith_b200")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 65408.0   # largest magnitude a cached value keeps (float16 parameters)
TINY = 1e-30      # rows or groups whose largest magnitude is below this quantise to zero


# ---------------------------------------------------------------------------
# cases
def listed():
    return [
        # the norm before a projection while four sequences decode
        dict(name="norm int8, 4 rows", op="norm", dtype="bf16", rows=4, cols=4096, out="int8",
             group=0),
        # the same in a prefill of a 4096-wide model
        dict(name="norm int8, 8192 rows", op="norm", dtype="f16", rows=8192, cols=4096,
             out="int8", group=0),
        # the widest residual stream, scales per 128 columns, an odd number of rows
        dict(name="norm e4m3, 16381 x 8192", op="norm", dtype="bf16", rows=16381, cols=8192,
             out="e4m3", group=128),
        # one new token of each of 64 sequences
        dict(name="cache, 64 tokens", op="cache", dtype="bf16", tokens=64, kv_heads=8, dim=128,
             group=32, page=64),
        # a prefill's keys and values, odd length, small pages
        dict(name="cache, 30011 tokens", op="cache", dtype="f16", tokens=30011, kv_heads=8,
             dim=128, group=32, page=16),
        # one sequence decodes at a short context: latency
        dict(name="attend 1 x 1021", op="attend", dtype="bf16", batch=1, queries=1, heads=32,
             kv_heads=8, dim=128, group=32, page=64, longest=1021, ragged=False),
        # a serving batch of ragged lengths, empty and one-token ones among them
        dict(name="attend 64 ragged to 4096", op="attend", dtype="f16", batch=64, queries=1,
             heads=32, kv_heads=8, dim=128, group=32, page=64, longest=4096, ragged=True),
        # several tokens are verified at once: seven heads share one, small head, small pages
        dict(name="attend 16 x 5 new tokens", op="attend", dtype="bf16", batch=16, queries=5,
             heads=14, kv_heads=2, dim=64, group=64, page=16, longest=2500, ragged=True),
        # long contexts
        dict(name="attend 8 x 65536", op="attend", dtype="bf16", batch=8, queries=1, heads=64,
             kv_heads=8, dim=128, group=128, page=128, longest=65536, ragged=False),
        # a projection of one token
        dict(name="product 1 x 4096 x 4096", op="product", x="bf16", dtype="bf16", rows=1,
             k=4096, n=4096, group=128, zeros=False),
        # the down projection fed by 8-bit activations, zero points, small groups
        dict(name="product e4m3 8 x 11008 x 4096", op="product", x="e4m3", dtype="bf16", rows=8,
             k=11008, n=4096, group=32, zeros=True),
        # the vocabulary's logits of a batch
        dict(name="product 16 x 4096 x 128256", op="product", x="f16", dtype="f16", rows=16,
             k=4096, n=128256, group=128, zeros=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "cache", "attend", "product"])
    if op == "norm":
        cols = rng.choice([_log(rng, 64, 20000), 8 * _log(rng, 16, 2048), 4096, 8192])
        rows = _log(rng, 1, max(1, min(40000, 16000 * 8192 // cols)))
        out = rng.choice(["int8", "e4m3"])
        # a row of int8 is read back by the per-row dequantisation
        group = 0 if out == "int8" else rng.choice([0, 32, 64, 128])
        # float32 rows only with e4m3: its own type has to absorb a flipped rounding
        dtype = rng.choice(["f16", "bf16"] if out == "int8" else ["f16", "bf16", "f32"])
        if dtype == "f32":
            rows = max(1, rows // 2)
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, out=out, group=group)
    if op == "cache":
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        return dict(op=op, dtype=rng.choice(["f16", "bf16"]),
                    tokens=_log(rng, 1, 30000 * 1024 // (dim * kv_heads)), kv_heads=kv_heads,
                    dim=dim, group=rng.choice([g for g in (32, 64, 128) if g <= dim]),
                    page=rng.choice([16, 32, 64, 128]))
    if op == "attend":
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        share = rng.choice([1, 2, 3, 4, 7, 8, 16])
        queries = rng.choice([1, 1, 1, 2, 4, _log(rng, 2, 64)])
        batch = _log(rng, 1, 64)
        # scores of the plain form: batch * heads * queries * longest
        most = min(7 * 65536 * 8 * 128 // (batch * kv_heads * dim),
                   300_000_000 // (batch * kv_heads * share * queries))
        longest = _log(rng, 1, max(1, min(100000, most)))
        return dict(op=op, dtype=rng.choice(["f16", "bf16"]), batch=batch, queries=queries,
                    heads=kv_heads * share, kv_heads=kv_heads, dim=dim,
                    group=rng.choice([g for g in (32, 64, 128) if g <= dim]),
                    page=rng.choice([16, 32, 64, 128]), longest=longest,
                    ragged=rng.random() < 0.5)
    k, n = _log(rng, 100, 16000), _log(rng, 100, 32000)
    n = min(n, 400_000_000 // k)
    rows = rng.choice([1, 1, 2, 4, 8, _log(rng, 1, 64)])
    x = rng.choice(["f16", "bf16", "f32", "int8", "e4m3"])
    return dict(op=op, x=x, dtype=x if x in DTYPES else rng.choice(["f16", "bf16"]), rows=rows,
                k=k, n=n, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)


def _lengths(case):
    """Tokens in the cache of each sequence, the new ones included."""
    batch, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * batch
    lens = [int(longest * (i + 1) / batch) for i in range(batch)]
    if batch > 2:
        lens[0], lens[1] = 0, min(1, longest)
    return lens


def work(case):
    op = case["op"]
    if op == "norm":
        m, n = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "f32" else 2
        scales = m * (-(-n // case["group"]) if case["group"] else 1)
        # x, residual and weight in, stream, 8-bit values and scales out; int8 is read back
        # in 16 bits
        back = 3 * m * n if case["out"] == "int8" else 0
        return {"bytes": 3 * m * n * size + n * size + m * n + 4 * scales + back,
                "flops": 8 * m * n}
    if op == "cache":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        held = values // 2 + 4 * values // case["group"]
        return {"bytes": 2 * values + held + held + 2 * values + 16 * case["tokens"],
                "flops": 6 * values}
    if op == "attend":
        dim, q = case["dim"], case["queries"]
        seen = sum(_lengths(case))
        pairs = sum(max(0, n - q + 1 + i) for n in _lengths(case) for i in range(q))
        held = seen * case["kv_heads"] * (dim + 8 * dim // case["group"])
        ends = 2 * 2 * case["batch"] * q * case["heads"] * dim
        return {"bytes": held + ends, "flops": 4 * pairs * case["heads"] * dim}
    m, k, n = case["rows"], case["k"], case["n"]
    scales = n * -(-k // case["group"]) * 2 * (2 if case["zeros"] else 1)
    size = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}[case["x"]]
    return {"bytes": n * k / 2 + scales + m * k * size + m * n * (4 if case["dtype"] == "f32" else 2),
            "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# layouts
def pack_nibbles(n):
    """Whole numbers 0..15 (last dimension even) as bytes, the earlier one in the low bits."""
    n = n.to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def unpack_nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def quantise(x, group):
    """Groups of the last dimension in 4 bits: (n, s, lo) with x near lo + n * s.
    s and lo are float16; n goes by their rounded values."""
    x = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, group))
    lo, hi = x.amin(-1), x.amax(-1)
    s, lo = ((hi - lo) / 15).half(), lo.half()
    step = s.float().unsqueeze(-1)
    n = torch.where(step > 0, ((x - lo.float().unsqueeze(-1)) / step).round().clamp(0, 15),
                    torch.zeros_like(x))
    return n.to(torch.uint8).flatten(-2), s, lo


def cache_bytes(k, v, group, page):
    """The cache's bytes for the tokens of every slot: k, v [pages * page, Hk, D] ->
    [pages, Hk, page / 16, 16 * (D + 8 * D / group)].  Each 16 tokens of one head lie
    together: the keys' 4-bit rows, their (s, lo), the values' rows, their (s, lo).  A
    row's 32-bit words hold eight dimensions each, in order for the values; for the keys
    word j of the row's quarter c holds dimensions 32 j + 8 c ... + 7."""
    slots, heads, dim = k.shape
    parts = []
    for x, is_key in ((k, True), (v, False)):
        n, s, lo = quantise(x, group)
        if is_key:
            n = n.view(slots, heads, dim // 32, 4, 8).transpose(2, 3).reshape(slots, heads, dim)
        rows = pack_nibbles(n)
        params = torch.stack((s, lo), -1).flatten(-2).view(torch.uint8)
        for part in (rows, params):
            part = part.reshape(slots // page, page // 16, 16, heads, part.shape[-1])
            parts.append(part.permute(0, 3, 1, 2, 4).flatten(-2))
    return torch.cat(parts, -1).contiguous()


def cache_views(data, dim, group):
    """The four fields of the cache's bytes, each as a view with a row for every token:
    data [..., Hk, page / 16, 16 * (D + 8 * D / group)] -> [..., page / 16, 16, Hk, bytes];
    the keys' rows, their (s, lo), the values' rows, their (s, lo)."""
    at, out = 0, []
    for size in 2 * (dim // 2, 4 * dim // group):
        field = data[..., at:at + 16 * size].unflatten(-1, (16, size))
        out.append(field.movedim(-4, -2))
        at += 16 * size
    return out


def token_values(rows, params, is_key, group):
    """Token rows of bytes and of (s, lo) as the float32 values that they stand for."""
    n = unpack_nibbles(rows)
    dim = n.shape[-1]
    if is_key:
        n = n.unflatten(-1, (4, dim // 32, 8)).transpose(-3, -2).flatten(-3)
    params = params.contiguous().view(torch.float16).unflatten(-1, (dim // group, 2)).float()
    y = n.unflatten(-1, (dim // group, group)) * params[..., :1] + params[..., 1:]
    return y.flatten(-2)


def weight_tiles(n, scales, zeros, group):
    """The product's weight layout: n [N, K] whole numbers 0..15, scales (and zeros)
    [N, ceil(K / group)] -> tiles [ceil(N / 16), ceil(K / 128), 16, 64] of bytes and
    [ceil(N / 16), ceil(K / 128), 128 / group, 16] of scales.  Word j of quarter c of a
    tile's row holds columns 32 j + 8 c ... + 7 of its 128."""
    rows, cols = n.shape
    nt, kt, gs = -(-rows // 16), -(-cols // 128), 128 // group
    n = torch.nn.functional.pad(n, (0, kt * 128 - cols, 0, nt * 16 - rows))
    n = n.view(nt, 16, kt, 4, 4, 8).permute(0, 2, 1, 4, 3, 5).reshape(nt, kt, 16, 128)
    out = [pack_nibbles(n).contiguous()]
    for t in (scales, zeros):
        if t is not None:
            t = torch.nn.functional.pad(t, (0, kt * gs - t.shape[1], 0, nt * 16 - rows))
            t = t.view(nt, 16, kt, gs).permute(0, 2, 3, 1).contiguous()
        out.append(t)
    return out


# ---------------------------------------------------------------------------
# inputs
def _activations(g, *shape):
    """Normal values with a few loud channels, as hidden states have them."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = torch.rand(shape[-1], generator=g, device="cuda") < 0.005
    return x * torch.where(loud, 20.0, 1.0)


def _keys(g, tokens, heads, dim):
    """Normal values around an offset of each channel, as keys have them."""
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda")
    return x + 2 * torch.randn((heads, dim), generator=g, device="cuda")


def _e4m3_rows(x):
    top = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * (448 / top)).clamp(-448, 448).to(torch.float8_e4m3fn), top / 448


def _int8_rows(x):
    top = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * (127 / top)).round().clamp(-127, 127).to(torch.int8), top / 127


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        import b200k
        s["b200k"] = b200k
    op = case["op"]
    if op == "norm":
        t = DTYPES[case["dtype"]]
        shape = (case["rows"], case["cols"])
        s["x"] = _activations(g, *shape).to(t)
        s["r"] = (3 * _activations(g, *shape)).to(t)
        s["w"] = (1 + 0.2 * torch.randn(shape[1], generator=g, device="cuda")).to(t)
    elif op == "cache":
        t, page = DTYPES[case["dtype"]], case["page"]
        tokens, heads, dim = case["tokens"], case["kv_heads"], case["dim"]
        s["k"] = _keys(g, tokens, heads, dim).to(t)
        s["v"] = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(t)
        # whole pages in the pool's order for a prefill; few tokens lie in a page each
        spread = tokens <= 256
        pages = (tokens if spread else -(-tokens // page)) + 3
        ids = torch.randperm(pages, generator=g, device="cuda")
        i = torch.arange(tokens, device="cuda")
        s["slots"] = ids[i] * page + i * 7 % page if spread else ids[i // page] * page + i % page
        dims = (pages, heads, page // 16, 16 * (dim + 8 * dim // case["group"]))
        s["data"] = torch.zeros(dims, dtype=torch.uint8, device="cuda")
        if own:  # the handle that names the bytes' geometry
            s["cache"] = b200k.KVCache4(s["data"], dim, case["group"])
    elif op == "attend":
        t, page = DTYPES[case["dtype"]], case["page"]
        heads, dim, lens = case["kv_heads"], case["dim"], _lengths(case)
        wide = max(1, -(-max(lens) // page))
        counts = torch.tensor([-(-n // page) for n in lens], device="cuda")
        pages = sum(-(-n // page) for n in lens) + 2
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        first = counts.cumsum(0) - counts
        j = torch.arange(wide, device="cuda")
        at = (first[:, None] + j).clamp(max=pages - 1)
        s["table"] = torch.where(j < counts[:, None], ids[at], -1).int().contiguous()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        offset = 2 * torch.randn((heads, dim), generator=g, device="cuda")
        s["data"] = torch.empty((pages, heads, page // 16, 16 * (dim + 8 * dim // case["group"])),
                                dtype=torch.uint8, device="cuda")
        part = max(1, (1 << 26) // (page * heads * dim))
        for p in range(0, pages, part):
            some = (min(part, pages - p) * page, heads, dim)
            k = torch.randn(some, generator=g, device="cuda") + offset
            v = torch.randn(some, generator=g, device="cuda")
            s["data"][p:p + part] = cache_bytes(k, v, case["group"], page)
        s["q"] = torch.randn((case["batch"], case["queries"], case["heads"], dim), generator=g,
                             device="cuda").to(t)
        if own:
            s["cache"] = b200k.KVCache4(s["data"], dim, case["group"])
    else:
        m, k, n, group = case["rows"], case["k"], case["n"], case["group"]
        groups = -(-k // group)
        q = torch.empty((n, k), dtype=torch.uint8, device="cuda")
        part = max(1, (1 << 27) // k)
        for i in range(0, n, part):
            w = torch.randn((min(part, n - i), k), generator=g, device="cuda")
            q[i:i + part] = (w * 2.7 + 8).round().clamp(0, 15).to(torch.uint8)
        scales = ((0.5 + torch.rand((n, groups), generator=g, device="cuda")) / (2.7 * k ** 0.5))
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(6, 11, (n, groups), generator=g, device="cuda").half()
        s["tiles"], s["scales"], s["zeros"] = weight_tiles(q, scales.half(), zeros, group)
        x, s["x_scale"] = _activations(g, m, k), None
        if case["x"] == "e4m3":
            s["x"], s["x_scale"] = _e4m3_rows(x)
        elif case["x"] == "int8":
            s["x"], s["x_scale"] = _int8_rows(x)
        else:
            s["x"] = x.to(DTYPES[case["x"]])
        if own:
            s["weight"] = b200k.W4Weight(s["tiles"], s["scales"], s["zeros"], n, k)
    return s


# ---------------------------------------------------------------------------
# one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_norm(s):
    b, case = s["b200k"], s["case"]
    int8 = case["out"] == "int8"
    h, q, scale = b.add_rmsnorm_quant(s["x"], s["r"], s["w"],
                                      dtype=torch.int8 if int8 else torch.float8_e4m3fn,
                                      group=case["group"] or None)
    return {"h": h, "q": b.dequant_int8(q, scale) if int8 else q, "scale": scale}


def _plain_norm(s):
    case = s["case"]
    h = (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * s["w"].float() * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)
    cols, group = case["cols"], case["group"] or case["cols"]
    groups = -(-cols // group)
    y = torch.nn.functional.pad(y, (0, groups * group - cols)).unflatten(-1, (groups, group))
    top = y.abs().amax(-1, keepdim=True)
    most = 127.0 if case["out"] == "int8" else 448.0
    fine = top >= TINY
    scale = torch.where(fine, top / most, torch.zeros_like(top))
    y = (y * torch.where(fine, most / top, torch.zeros_like(top))).clamp(-most, most)
    if case["out"] == "int8":
        q = (y.round() * scale).flatten(-2)[..., :cols].half()
    else:
        q = y.flatten(-2)[..., :cols].to(torch.float8_e4m3fn)
    return {"h": h, "q": q, "scale": scale.squeeze(-1)}


def _own_cache(s):
    b = s["b200k"]
    b.kv_cache_write(s["cache"], s["k"], s["v"], s["slots"])
    k, v = b.kv_cache_read(s["cache"], s["slots"], dtype=s["k"].dtype)
    return {"k": k, "v": v}


def _plain_cache(s):
    case, slots = s["case"], s["slots"]
    dim, group, page = case["dim"], case["group"], case["page"]
    at = slots // page, slots % page // 16, slots % 16
    views = cache_views(s["data"], dim, group)
    out = []
    for name, is_key in (("k", True), ("v", False)):
        rows, params = views[:2] if is_key else views[2:]
        n, step, lo = quantise(s[name], group)
        if is_key:
            n = n.unflatten(-1, (dim // 32, 4, 8)).transpose(-3, -2).flatten(-3)
        rows[at] = pack_nibbles(n)
        params[at] = torch.stack((step, lo), -1).flatten(-2).view(torch.uint8)
        out.append(token_values(rows[at], params[at], is_key, group).to(s[name].dtype))
    return {"k": out[0], "v": out[1]}


def _own_attend(s):
    return s["b200k"].cache_attention(s["q"], s["cache"], s["table"], s["lens"])


def _plain_attend(s):
    case, q = s["case"], s["q"]
    dim, group, hk = case["dim"], case["group"], case["kv_heads"]
    batch, queries, heads = q.shape[:3]
    views = cache_views(s["data"][s["table"].clamp(min=0).long()], dim, group)
    kv = [token_values(rows, params, is_key, group).flatten(1, 3).transpose(1, 2)  # [B, Hk, L, D]
          for rows, params, is_key in ((*views[:2], True), (*views[2:], False))]
    share = heads // hk
    f = q.float().view(batch, queries, hk, share, dim).permute(0, 2, 3, 1, 4)
    f = f.reshape(batch, hk, share * queries, dim)
    scores = torch.matmul(f, kv[0].transpose(-1, -2)) * dim ** -0.5
    j = torch.arange(scores.shape[-1], device=q.device)
    last = s["lens"][:, None] - queries + torch.arange(queries, device=q.device)  # [B, Sq]
    seen = (j <= last[..., None])[:, None, None]                                  # [B, 1, 1, Sq, L]
    scores = scores.view(batch, hk, share, queries, -1).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, hk, share * queries, -1), kv[1])
    o = o.view(batch, hk, share, queries, dim) / total.masked_fill(total == 0, 1)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim).to(q.dtype)


def _own_product(s):
    return s["b200k"].w4_matmul(s["x"], s["weight"], x_scale=s["x_scale"],
                                out_dtype=DTYPES[s["case"]["dtype"]])


def _plain_product(s):
    case = s["case"]
    k, n, group = case["k"], case["n"], case["group"]
    w = unpack_nibbles(s["tiles"]).unflatten(-1, (4, 4, 8)).transpose(-3, -2)
    w = w.reshape(*w.shape[:3], 128 // group, group).float()     # [nt, kt, 16, gs, group]
    scales = s["scales"].float().transpose(2, 3).unsqueeze(-1)   # [nt, kt, 16, gs, 1]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().transpose(2, 3).unsqueeze(-1)
    w = ((w - zeros) * scales).flatten(-2).transpose(1, 2).reshape(w.shape[0] * 16, -1)[:n, :k]
    x = s["x"].float()
    if s["x_scale"] is not None:
        x = x * s["x_scale"]
    return torch.matmul(x, w.t()).to(DTYPES[case["dtype"]])


_own = {"norm": _own_norm, "cache": _own_cache, "attend": _own_attend, "product": _own_product}
_plain = {"norm": _plain_norm, "cache": _plain_cache, "attend": _plain_attend,
          "product": _plain_product}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one row, token, sequence or tile row at a time
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "cache": _exact_cache, "attend": _exact_attend,
            "product": _exact_product}[case["op"]](case, s)


def _near_e4m3(y):
    """y rounded to the nearest value of three fraction bits, at least 2^-9 apart."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e - 4, min=-9))
    return (y / step).round() * step


def _exact_norm(case, s):
    h = (s["x"].double() + s["r"].double()).to(s["x"].dtype)
    w, cols = s["w"].double(), case["cols"]
    most = 127.0 if case["out"] == "int8" else 448.0
    qs, scales = [], []
    part = max(1, (1 << 25) // cols)
    for i in range(0, case["rows"], part):
        f = h[i:i + part].double()
        y = f * w / torch.sqrt((f * f).sum(1, keepdim=True) / cols + 1e-6)
        q, sc = torch.empty_like(y), []
        for a in range(0, cols, case["group"] or cols):
            z = y[:, a:a + (case["group"] or cols)]
            top = z.abs().amax(1, keepdim=True)
            unit = torch.where(top < TINY, torch.ones_like(top), top / most)
            if case["out"] == "int8":
                q[:, a:a + z.shape[1]] = (z / unit).round() * unit
            else:
                q[:, a:a + z.shape[1]] = _near_e4m3(z / unit)
            sc.append(torch.where(top < TINY, torch.zeros_like(top), unit))
        qs.append(q.float())
        scales.append(torch.cat(sc, 1))
    return {"h": h.double(), "q": torch.cat(qs).double(), "scale": torch.cat(scales)}


def _exact_cache(case, s):
    out = {}
    for name in ("k", "v"):
        x = s[name].double().clamp(-LIMIT, LIMIT)
        y = torch.empty_like(x)
        for a in range(0, case["dim"], case["group"]):
            z = x[..., a:a + case["group"]]
            lo, hi = z.amin(-1, keepdim=True), z.amax(-1, keepdim=True)
            step, lo = ((hi - lo) / 15).half().double(), lo.half().double()
            n = ((z - lo) / torch.where(step > 0, step, torch.ones_like(step))).round()
            y[..., a:a + case["group"]] = lo + step * n.clamp(0, 15)
        out[name] = y
    return out


def _token_rows(data, dim, group, is_key):
    """The values of one head's micro blocks [m, bytes], in 64 bits: [16 m, D]."""
    half = 8 * dim + 64 * dim // group
    block = data[:, :half] if is_key else data[:, half:]
    rows = block[:, :8 * dim].reshape(-1, dim // 2).long()
    params = block[:, 8 * dim:].contiguous().view(torch.float16).double().reshape(-1, dim // group, 2)
    d = torch.arange(dim, device=data.device)
    if is_key:   # where dimension d lies among the row's nibbles
        place = d % 32 // 8 * (dim // 4) + d // 32 * 8 + d % 8
    else:
        place = d
    n = (rows[:, place // 2] >> (4 * (place % 2))) & 15
    return params[:, d // group, 0] * n + params[:, d // group, 1]


def _exact_attend(case, s):
    if sum(_lengths(case)) * case["kv_heads"] * case["dim"] > 6e8:
        return None
    dim, group, q = case["dim"], case["group"], s["q"].double()
    batch, queries, heads = q.shape[:3]
    share, o = heads // case["kv_heads"], torch.zeros_like(q)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        blocks = s["data"][s["table"][b, :-(-n // case["page"])].long()]
        for head in range(case["kv_heads"]):
            data = blocks[:, head].flatten(0, 1)
            k = _token_rows(data, dim, group, True)[:n]
            v = _token_rows(data, dim, group, False)[:n]
            for i in range(max(0, queries - n), queries):
                m = n - queries + i + 1
                z = q[b, i, head * share:(head + 1) * share] @ k[:m].T / math.sqrt(dim)
                o[b, i, head * share:(head + 1) * share] = torch.softmax(z, -1) @ v[:m]
    return o


def _exact_product(case, s):
    k, n, group = case["k"], case["n"], case["group"]
    x = s["x"].double()
    if s["x_scale"] is not None:
        x = x * s["x_scale"].double()
    tiles = s["tiles"]
    y = torch.zeros((x.shape[0], tiles.shape[0] * 16), dtype=torch.float64, device=x.device)
    for kt in range(tiles.shape[1]):
        for j in range(4):                       # columns 32 j ... + 31 of the 128
            a = 128 * kt + 32 * j
            if a >= k:
                break
            cols = torch.arange(min(32, k - a), device=x.device)
            place = cols // 8 * 32 + 8 * j + cols % 8
            w = (tiles[:, kt][:, :, place // 2].long() >> (4 * (place % 2))) & 15
            scale = s["scales"][:, kt, 32 * j // group].double().unsqueeze(-1)
            zero = 8.0 if s["zeros"] is None else s["zeros"][:, kt, 32 * j // group].double().unsqueeze(-1)
            w = ((w.double() - zero) * scale).flatten(0, 1)
            y += x[:, a:a + len(cols)] @ w.T
    return y[:, :n]
