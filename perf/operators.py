"""Cases of the operators around the 8-bit KV cache: writing it (RoPE + quantise + append of a ragged batch), reading
it back to 16 bits, and attention over it -- one token per sequence, and ragged chunks of new tokens, both with an
optional sliding window and always-visible first tokens.

A cache row (one position of one KV head, 128 elements) is held as 128 e4m3 codes and one exponent byte x:
value = code * 2^(x - 127).  The exponent is the smallest for which the row's largest magnitude is at most 448 steps.

`run` is the operators in elementary torch operations where `own` is false, and this package's calls where it is true.
"""
import math

import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases
def _case(name, kind, dtype, H, kvH, B, ctx, new=(0, 0), layout="paged", page=256, neox=True, window=0, sink=0):
    c = {"kind": kind, "dtype": dtype, "H": H, "kvH": kvH, "B": B, "ctx_min": ctx[0], "ctx_max": ctx[1],
         "new_min": new[0], "new_max": new[1], "layout": layout, "page": page, "neox": neox, "window": window,
         "sink": sink}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the K/V write of a decode step of a served batch: one new token for each of 64 sequences
        _case("write_step", "write", "bf16", 40, 8, 64, (300, 4000), (1, 1)),
        # prompts of different lengths enter the cache together, some of them behind a cached prefix
        _case("write_prompts", "write", "bf16", 40, 8, 12, (0, 2000), (37, 3900)),
        # multi-head model with interleaved pairs and a flat token-major cache, the reference's layout
        _case("write_flat_mha", "write", "fp16", 40, 40, 8, (0, 700), (129, 2048), layout="token", neox=False),
        # a cached prefix goes back to 16 bits for a path that works on 16-bit caches
        _case("read_prefix", "read", "bf16", 40, 8, 6, (9000, 32768)),
        # the same for a short prompt of a small model
        _case("read_short", "read", "fp16", 12, 2, 3, (60, 511), page=64),
        # one sequence of a small model, a few hundred cached tokens: latency
        _case("decode_one", "decode", "bf16", 12, 2, 1, (511, 511), page=64),
        # a served batch at ordinary lengths
        _case("decode_batch", "decode", "bf16", 40, 8, 64, (300, 4096)),
        # long contexts, every one of another length: the largest read of the cache
        _case("decode_long", "decode", "fp16", 40, 8, 48, (3000, 32768)),
        # window of 4096 and four first tokens over long caches, whose other pages a server has given back
        _case("decode_window", "decode", "bf16", 40, 8, 64, (2000, 32768), window=4096, sink=4),
        # several tokens per sequence at once: a draft being checked
        _case("chunk_draft", "chunk", "bf16", 12, 2, 4, (200, 1500), (2, 5), page=64),
        # prompts of different lengths behind cached prefixes, with a window
        _case("chunk_ragged", "chunk", "fp16", 40, 8, 6, (100, 5000), (33, 1024), page=128, window=2048, sink=4),
        # a chunk of 4096 tokens of a long prompt
        _case("chunk_long", "chunk", "bf16", 40, 8, 1, (12288, 12288), (4096, 4096)),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk"])
    H, kvH = rng.choice([(40, 8), (40, 40), (12, 2), (28, 4), (16, 16), (8, 1), (14, 2), (32, 2)])
    dtype, layout, neox = rng.choice(["bf16", "fp16"]), rng.choice(["paged", "paged", "head", "token"]), rng.random() < 0.5
    page = rng.choice([64, 128, 256])
    window, sink = (0, 0) if rng.random() < 0.5 else (_spread(rng, 1, 8192), rng.choice([0, 1, 4, 64, 130]))
    if kind in ("write", "read"):
        top = 60000 if kind == "write" else 120000       # tokens of a model of eight heads
        B = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, min(8192, top * 8 // (H + kvH * 2) // B)))
        ctx = _spread(rng, 1, 4096)
        if kind == "read":
            return _case(None, kind, dtype, H, kvH, B, (max(0, new // 3), new), (0, 0), layout, page, neox)
        return _case(None, kind, dtype, H, kvH, B, (rng.choice([0, ctx // 2]), ctx), (max(1, new // rng.choice([1, 2, 9])), new),
                     layout, page, neox)
    if kind == "decode":
        B = _spread(rng, 1, 64)
        ctx = _spread(rng, 1, max(2, min(32768, 6000000 // (B * kvH))))
        return _case(None, kind, dtype, H, kvH, B, (rng.choice([0, ctx // 9, ctx]), ctx), (0, 0), layout, page, neox, window, sink)
    B = _spread(rng, 1, 16)
    new = _spread(rng, 1, 2048)
    ctx = _spread(rng, 1, max(2, min(16384, 300000000 // (B * new * H) * 4)))
    return _case(None, kind, dtype, H, kvH, B, (rng.choice([0, ctx // 2]), ctx), (max(1, new // rng.choice([1, 3, 20])), new),
                 layout, page, neox, window, sink)


def _lens(lo, hi, B):
    """B lengths from lo to hi in no order; the longest and the shortest are among them."""
    if B == 1:
        return [hi]
    golden = 0.6180339887498949
    got = [lo + int((hi - lo) * ((0.3 + b * golden) % 1.0)) for b in range(B)]
    got[B // 2], got[-1] = hi, lo
    return got


def _shape(case):
    """Cached tokens before the call, and new tokens, of every sequence."""
    ctx = _lens(case["ctx_min"], case["ctx_max"], case["B"])
    new = _lens(case["new_min"], case["new_max"], case["B"])[::-1]
    if case["kind"] == "read":
        return [0] * case["B"], ctx
    if case["kind"] == "decode":
        return ctx, [0] * case["B"]
    return ctx, new


def _first_visible(pos, window):
    return max(0, pos - window + 1) if window else 0


def work(case):
    H, kvH, win, sink = case["H"], case["kvH"], case["window"], case["sink"]
    ctx, new = _shape(case)
    row = kvH * (D + 1) * 2                              # one position of the cache, K and V with their exponents
    total = sum(new)
    if case["kind"] == "write":
        spans, table_rows, end = sorted((c, c + n) for c, n in zip(ctx, new)), 0, 0
        for a, b in spans:
            table_rows += max(0, b - max(a, end))
            end = max(end, b)
        in_out = total * (2 * H + 2 * 2 * kvH) * D * 2   # q, k, v in; q, and k and v as read back, out
        return {"bytes": in_out + total * row + table_rows * D * 4, "flops": total * (H + kvH) * D * 3}
    if case["kind"] == "read":
        return {"bytes": total * (row + 2 * kvH * D * 2), "flops": total * 2 * kvH * D}
    if case["kind"] == "decode":
        seen = 0
        for c in ctx:
            lo = _first_visible(c - 1, win)
            seen += c - lo + min(sink, lo) if c else 0
        return {"bytes": seen * row + 2 * case["B"] * H * D * 2, "flops": 4.0 * D * H * seen}
    pairs, touched = 0, 0
    for c, n in zip(ctx, new):
        for pos in range(c, c + n):
            lo = _first_visible(pos, win)
            pairs += pos + 1 - lo + min(sink, lo)
        if n:
            lo = _first_visible(c, win)
            touched += c + n - lo + min(sink, lo)
    return {"bytes": touched * row + 2 * total * H * D * 2, "flops": 4.0 * D * H * pairs}


# ---------------------------------------------------------------------------------------------- quantiser
def _pow2(e):
    """2^e in fp32 for whole e in -126 .. 127, from the bit pattern."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 [..., 128] -> e4m3 codes as bytes, exponent bytes [...]."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)                             # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -100)).clamp_(min=-100)
    codes = (x * _pow2(-e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, exps):
    return codes.view(torch.float8_e4m3fn).to(torch.float32).mul_(_pow2(exps.to(torch.int32) - 127)[..., None])


# ---------------------------------------------------------------------------------------------- state
def _cache(case, capacity, gen, filled, dev):
    """Codes and exponents of K and V in the case's layout, and the page table."""
    B, kvH = case["B"], case["kvH"]
    if case["layout"] == "paged":
        ps = case["page"]
        per = (capacity + ps - 1) // ps
        n = B * per + 3
        table = torch.randperm(n, generator=gen, device=dev)[: B * per].reshape(B, per).to(torch.int32)
        lead = (n, kvH, ps)
    else:
        capacity = (capacity + 63) // 64 * 64
        table = None
        lead = (B, kvH, capacity)                        # the token-major cache is a transposed view of [B, capacity, kvH]
    got = []
    for is_v in (False, True):
        if filled:
            codes = torch.empty(lead + (D,), dtype=torch.uint8, device=dev)
            exps = torch.empty(lead, dtype=torch.uint8, device=dev)
            step = max(1, (1 << 27) // (kvH * lead[2] * D))
            for i in range(0, lead[0], step):
                part = (min(step, lead[0] - i),) + lead[1:]
                x = torch.randn(part + (D,), generator=gen, device=dev)
                x *= torch.exp(0.4 * torch.randn(part + (1,), generator=gen, device=dev))       # tokens differ in size
                if not is_v:                             # a few channels of K are much larger than the others
                    x *= 1.0 + 4.0 * (torch.rand(part[:2] + (1, D), generator=gen, device=dev) < 0.03)
                codes[i:i + step], exps[i:i + step] = _quantise(x)
        else:
            codes = torch.zeros(lead + (D,), dtype=torch.uint8, device=dev)
            exps = torch.full(lead, 127, dtype=torch.uint8, device=dev)
        if case["layout"] == "token":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
        got += [codes, exps]
    return got, table, (table.shape[1] * case["page"] if table is not None else capacity)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, H, kvH = case["B"], case["H"], case["kvH"]
    ctx, new = _shape(case)
    capacity = max(1, max(c + n for c, n in zip(ctx, new)))
    (k, kx, v, vx), table, max_pos = _cache(case, capacity, gen, case["kind"] != "write", dev)
    s = {"case": case, "k": k, "kx": kx, "v": v, "vx": vx, "table": table, "max_pos": max_pos,
         "total": sum(new), "max_new": max(new), "max_len": capacity,
         "lens": torch.tensor(ctx, dtype=torch.int32, device=dev),
         "tok": torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)}
    tokens = B if case["kind"] == "decode" else sum(new)

    def rows(heads, scale=1.0):
        return (torch.randn(tokens, heads, D, generator=gen, device=dev) * scale).to(dt)

    if case["kind"] == "write":
        s["q"], s["knew"], s["vnew"] = rows(H), rows(kvH, 2.0), rows(kvH)
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))
        angle = torch.arange(max_pos, device=dev, dtype=torch.float64)[:, None] * inv
        s["freqs"] = torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).contiguous()
    elif case["kind"] != "read":
        s["q"] = rows(H)
    if case["kind"] == "read":
        s["kout"], s["vout"] = rows(kvH), rows(kvH)
    else:
        s["out"] = torch.zeros(tokens, H, D, dtype=dt, device=dev)
        if case["kind"] == "write":
            s["kout"], s["vout"] = torch.zeros_like(s["knew"]), torch.zeros_like(s["vnew"])
    return s


# ---------------------------------------------------------------------------------------------- this package's calls
def _handles(s):
    """The descriptors and the workspace that a program makes once for its cache."""
    if "ops" in s:
        return s["ops"]
    from llm_simple_b200 import ops
    case = s["case"]
    B, H, kvH = case["B"], case["H"], case["kvH"]
    dt = ops.DT_BFLOAT16 if case["dtype"] == "bf16" else ops.DT_FLOAT16
    paged = case["layout"] == "paged"
    desc = ops.make_desc(dt, B, H, kvH, 1, case["page"] if paged else s["max_pos"],
                         layout="token" if case["layout"] == "token" else "head", is_neox=case["neox"])
    pages = ops.make_pages(s["table"], case["page"], kvH * case["page"] * D, s["k"].shape[0]) if paged else None
    kv = ops.make_kv_q8(s["k"], s["v"], s["kx"], s["vx"], s["max_pos"])
    ws, n = None, 0
    if case["kind"] == "decode":
        n = ops.gpu_attn_decode_q8_workspace_bytes(desc, max(1, s["max_len"]))
    elif case["kind"] == "chunk":
        n = ops.gpu_attn_chunk_q8_workspace_bytes(desc, s["total"], s["max_new"], s["max_len"])
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=s["k"].device)
    s["ops"] = (ops, desc, pages, kv, ws, n)
    return s["ops"]


def _run_own(s):
    ops, desc, pages, kv, ws, n = _handles(s)
    case = s["case"]
    if case["kind"] == "write":
        ops.gpu_rope_kv_append_q8_layer(desc, pages, kv, s["out"], s["q"], s["knew"], s["vnew"], s["freqs"], s["tok"],
                                        s["lens"], s["total"])
        ops.gpu_kv_read_q8_layer(desc, pages, kv, s["kout"], s["vout"], s["tok"], s["lens"], s["total"])
        return [s["out"], s["kout"], s["vout"]]
    if case["kind"] == "read":
        ops.gpu_kv_read_q8_layer(desc, pages, kv, s["kout"], s["vout"], s["tok"], None, s["total"])
        return [s["kout"], s["vout"]]
    if case["kind"] == "decode":
        ops.gpu_attn_decode_q8_layer(desc, pages, kv, s["out"], s["q"], s["lens"], s["max_len"], case["window"],
                                     case["sink"], ws, n)
    else:
        ops.gpu_attn_chunk_q8_layer(desc, pages, kv, s["out"], s["q"], s["tok"], s["lens"], s["total"], s["max_new"],
                                    s["max_len"], case["window"], case["sink"], ws, n)
    return [s["out"]]


# ---------------------------------------------------------------------------------------------- plain forms
def _token_index(s):
    """Sequence, row within the sequence, and cache position of every new token."""
    counts = (s["tok"][1:] - s["tok"][:-1]).long()
    b = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts, output_size=s["total"])
    r = torch.arange(s["total"], device=counts.device) - s["tok"].long()[b]
    start = s["lens"].long()[b] if s["case"]["kind"] != "read" else 0
    return b, r, start + r


def _rotate(x, cs, neox):
    """fp32 rows [tokens, heads, 128] by the table rows [tokens, 64, 2]."""
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    if neox:
        a, b = x[..., :64], x[..., 64:]
        return torch.cat([a * c - b * n, a * n + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)


def _slots(s, b, pos):
    """Index of (sequence, position) in the caches' first and third dimensions."""
    if s["table"] is None:
        return b, pos
    ps = s["case"]["page"]
    return s["table"].long()[b, pos // ps], pos % ps


def _read(s, b, pos):
    i, j = _slots(s, b, pos)
    return _values(s["k"][i, :, j], s["kx"][i, :, j]), _values(s["v"][i, :, j], s["vx"][i, :, j])


def _whole(s, codes, exps):
    """The cache of every sequence in fp32, [batch][kv head][max_len][128]."""
    if s["table"] is None:
        return _values(codes[:, :, : s["max_len"]], exps[:, :, : s["max_len"]])
    t = s["table"].long()
    B, per = t.shape
    c = codes[t].transpose(1, 2).reshape(B, codes.shape[1], -1, D)[:, :, : s["max_len"]]
    x = exps[t].transpose(1, 2).reshape(B, codes.shape[1], -1)[:, :, : s["max_len"]]
    return _values(c, x)


def _attend(s, q, pos, live):
    """fp32 q [batch][rows][H][128]; pos [batch][rows] the rows' positions; live: the rows that exist."""
    case = s["case"]
    B, m, H = q.shape[:3]
    kvH = case["kvH"]
    g = H // kvH
    col = torch.arange(s["max_len"], device=q.device)
    seen = col <= pos[..., None]
    if case["window"]:
        seen &= (col > pos[..., None] - case["window"]) | (col < case["sink"])
    seen &= live[..., None]
    k = _whole(s, s["k"], s["kx"])
    x = torch.matmul(q.reshape(B, m, kvH, g, D).permute(0, 2, 3, 1, 4).reshape(B, kvH, g * m, D), k.transpose(2, 3))
    del k
    x = x.reshape(B, kvH, g, m, -1).mul_(1.0 / math.sqrt(D))
    hidden = ~seen[:, None, None]
    top = x.masked_fill_(hidden, -math.inf).amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = _whole(s, s["v"], s["vx"])
    v.masked_fill_(~seen.any(1)[:, None, :, None], 0.0)
    o = torch.matmul(x.reshape(B, kvH, g * m, -1), v).reshape(B, kvH, g, m, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, m, H, D)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "write":
        b, _, pos = _token_index(s)
        cs = s["freqs"][pos]
        s["out"].copy_(_rotate(s["q"].float(), cs, case["neox"]))
        i, j = _slots(s, b, pos)
        s["k"][i, :, j], s["kx"][i, :, j] = _quantise(_rotate(s["knew"].float(), cs, case["neox"]))
        s["v"][i, :, j], s["vx"][i, :, j] = _quantise(s["vnew"].float())
        k, v = _read(s, b, pos)
        s["kout"].copy_(k)
        s["vout"].copy_(v)
        return [s["out"], s["kout"], s["vout"]]
    if case["kind"] == "read":
        b, _, pos = _token_index(s)
        k, v = _read(s, b, pos)
        s["kout"].copy_(k)
        s["vout"].copy_(v)
        return [s["kout"], s["vout"]]
    if case["kind"] == "decode":
        pos = s["lens"].long()[:, None] - 1
        s["out"].copy_(_attend(s, s["q"].float()[:, None], pos, pos >= 0)[:, 0])
        return [s["out"]]
    b, r, pos = _token_index(s)
    m = s["max_new"]
    q = torch.zeros(case["B"], m, case["H"], D, device=s["q"].device)
    q[b, r] = s["q"].float()
    rows = torch.arange(m, device=b.device)
    live = rows < (s["tok"][1:] - s["tok"][:-1]).long()[:, None]
    s["out"].copy_(_attend(s, q, s["lens"].long()[:, None] + rows, live)[b, r])
    return [s["out"]]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_rotate(x, row, neox):
    c, n = row[..., 0].double(), row[..., 1].double()
    z = torch.view_as_complex(torch.stack([x[..., :64], x[..., 64:]], -1) if neox else x.unflatten(-1, (64, 2)).contiguous())
    z = z * torch.complex(c, n)[:, None]
    return torch.cat([z.real, z.imag], -1) if neox else torch.view_as_real(z).flatten(-2)


def _exact_cells(x):
    """What the cache stands for after rows x (fp64) were written."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(min=-100.0)
    scale = torch.exp2(e.round())
    y = x / scale
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)     # spacing of e4m3 there
    return torch.round(y / unit) * unit * scale


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _shape(case)
    B, H, kvH = case["B"], case["H"], case["kvH"]
    dev = s["k"].device

    def row_values(codes, exps, b, pos):
        """fp64 [positions][kv heads][128] of one sequence."""
        if s["table"] is not None:
            at = s["table"][b].long()[pos // case["page"]]
            c, x = codes[at, :, pos % case["page"]], exps[at, :, pos % case["page"]]
        else:
            c, x = codes[b].transpose(0, 1)[pos], exps[b].transpose(0, 1)[pos]
        return c.view(torch.float8_e4m3fn).double() * torch.exp2(x.double() - 127.0)[..., None]

    if case["kind"] == "write":
        pos = torch.cat([torch.arange(c, c + n, device=dev) for c, n in zip(ctx, new)])
        row = s["freqs"][pos]
        return [_exact_rotate(s["q"].double(), row, case["neox"]),
                _exact_cells(_exact_rotate(s["knew"].double(), row, case["neox"])), _exact_cells(s["vnew"].double())]
    if case["kind"] == "read":
        got = [[row_values(s[c], s[x], b, torch.arange(n, device=dev)) for b, n in enumerate(new)]
               for c, x in (("k", "kx"), ("v", "vx"))]
        return [torch.cat(p) for p in got]
    g = H // kvH
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    at = 0
    for b in range(B):
        first, rows = (ctx[b] - 1, 1) if case["kind"] == "decode" else (ctx[b], new[b])
        last = first + rows
        if last > 0:
            span = torch.arange(last, device=dev)
            mine = torch.arange(first, last, device=dev)[:, None]
            hidden = span > mine
            if case["window"]:
                hidden |= (span <= mine - case["window"]) & (span >= case["sink"])
            k, v = row_values(s["k"], s["kx"], b, span), row_values(s["v"], s["vx"], b, span)
            for j in range(H):
                score = (s["q"][at:at + rows, j].double() @ k[:, j // g].T) / math.sqrt(D)
                out[at:at + rows, j] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, j // g]
        at += rows
    return [out]
