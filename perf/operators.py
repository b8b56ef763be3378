"""Workloads of the cache-compression operators: a KV cache held in 4 bits (append, read-back, decode and chunked
prefill attention) and eviction by accumulated attention weight (accumulation over the queries, selection and
compaction).

``run`` computes each in its plain form -- elementary torch operations on fp32 -- or, where ``own`` is set, through
the calls a user of b2pa makes.  Sizes follow the serving configurations of this repository: 64 sequences of 128 to
1024 tokens with 8 heads of 64 channels (fp32), prompt chunks of 256 tokens on prefixes of up to 768, and sequences of
1024 to 8192 tokens with 32 heads of 128 channels (bf16).

The 4-bit format.  A row of D channels is cut into groups of 16.  Each group has a scale s, an unsigned 8-bit float
with 5 exponent and 3 mantissa bits (the byte shifted left by 7 is the fp16 number), and 16 codes c = round(x / s) in
-7..7, stored as c + 8 in a nibble; s is max|x| / 7 rounded to nearest even, at most 9216.  A group with a NaN or an
infinity stores the NaN scale 255.  A page of one head holds the codes [block_size, D / 2] (even channel in the low
nibble), then the scales: [block_size, D / 16] in the K pool, [D / 16, block_size] in the V pool.  Pools are uint8
[blocks, H, block_size, D * 9 / 16].
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _b2pa():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "efficient-inference-system_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2pa

    return b2pa


# --------------------------------------------------------------------- cases
def listed():
    return [
        # the append of one decode step of 64 requests: the smallest call, once per layer and token
        {"name": "append-step", "op": "append", "dtype": "f32", "B": 64, "H": 8, "D": 64, "bs": 16, "T": 1, "lo": 128,
         "hi": 1024},
        # a batch of ragged prompts going into the cache whole
        {"name": "append-prompts", "op": "append", "dtype": "bf16", "B": 8, "H": 32, "D": 128, "bs": 16, "T": 1531,
         "lo": 0, "hi": 37},
        # the decode step of a batch of short requests (fp32 model, 8 heads of 64)
        {"name": "decode-short", "op": "decode", "dtype": "f32", "B": 64, "H": 8, "D": 64, "bs": 16, "lo": 128,
         "hi": 1024},
        # one request alone on the GPU with a long context: few rows, a long axis
        {"name": "decode-alone", "op": "decode", "dtype": "bf16", "B": 1, "H": 32, "D": 128, "bs": 16, "lo": 8001,
         "hi": 8001},
        # one GPU's share (64 of 512) of the large serving batch
        {"name": "decode-long", "op": "decode", "dtype": "bf16", "B": 64, "H": 32, "D": 128, "bs": 16, "lo": 1024,
         "hi": 8192},
        # chunked prefill of the fp32 model: 256-token chunks on cached prefixes
        {"name": "prefill-chunk", "op": "prefill", "dtype": "f32", "B": 8, "H": 8, "D": 64, "bs": 16, "T": 256, "lo": 0,
         "hi": 768},
        # the last chunk of two long prompts (bf16 model), an odd chunk length
        {"name": "prefill-long", "op": "prefill", "dtype": "bf16", "B": 2, "H": 32, "D": 128, "bs": 16, "T": 1021,
         "lo": 1024, "hi": 7168},
        # a decode step's weights added to the running sums, 16-bit cache
        {"name": "weights-step", "op": "weights", "dtype": "bf16", "cache": "plain", "B": 32, "H": 32, "D": 128,
         "bs": 16, "T": 1, "window": 0, "lo": 1024, "hi": 8192},
        # a prompt chunk's weights, fp32 cache: every query counts
        {"name": "weights-chunk", "op": "weights", "dtype": "f32", "cache": "plain", "B": 8, "H": 8, "D": 64, "bs": 16,
         "T": 256, "window": 0, "lo": 0, "hi": 768},
        # the last 64 queries of long prompts rank a 4-bit cache's tokens
        {"name": "weights-window", "op": "weights", "dtype": "f16", "cache": "kv4", "B": 4, "H": 32, "D": 128, "bs": 16,
         "T": 500, "window": 64, "lo": 1024, "hi": 7168},
        # a batch of short requests cut to a budget, fp32 cache
        {"name": "evict-short", "op": "evict", "dtype": "f32", "cache": "plain", "B": 64, "H": 8, "D": 64, "bs": 16,
         "keep": 200, "recent": 50, "lo": 128, "hi": 1024},
        # long contexts cut to a quarter, 16-bit cache
        {"name": "evict-long", "op": "evict", "dtype": "bf16", "cache": "plain", "B": 8, "H": 32, "D": 128, "bs": 16,
         "keep": 2048, "recent": 256, "lo": 4096, "hi": 8192},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    op = rng.choice(["append", "decode", "prefill", "weights", "evict"])
    case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "H": rng.choice([1, 2, 3, 5, 8, 12, 16, 32]),
            "D": rng.choice([64, 64, 128, 128, 256]), "bs": rng.choice([8, 16, 16, 32])}
    if op == "append":
        case["T"] = spread(1, 1500)
        case["B"] = spread(1, max(1, min(64, 12000 // case["T"])))
        case["lo"], case["hi"] = 0, spread(1, 500)
        return case
    if op == "decode":
        case["hi"] = spread(1, 16000)
        case["B"] = spread(1, 64)
        room = 64 * 8192 * 32 * 128 // (case["H"] * case["D"])
    elif op == "evict":
        case["cache"] = rng.choice(["plain", "kv4"])
        case["hi"] = spread(2, 8192)
        case["B"] = spread(1, 64)
        room = 8 * 8192 * 32 * 128 * SIZE["bf16"] // (case["H"] * case["D"] * SIZE[case["dtype"]])
    else:
        case["T"] = spread(2, 1000) if op == "prefill" else rng.choice([1, spread(2, 600)])
        case["hi"] = spread(1, 7000)
        case["B"] = spread(1, 16)
        # the fp32 products cost several times the 16-bit ones
        most = 2 ** 31 if case["dtype"] == "f32" else 2 ** 35
        room = most // (case["H"] * case["D"] * case["T"])
        if op == "weights":
            case["cache"] = rng.choice(["plain", "kv4"])
            case["window"] = rng.choice([0, 0, 1, spread(1, case["T"])])
    case["hi"] = max(2, min(case["hi"], room // max(1, min(case["B"], room // 64 + 1))))
    case["B"] = max(1, min(case["B"], room // case["hi"]))
    case["lo"] = rng.choice([0 if op == "prefill" else 1, case["hi"] // 8, case["hi"]])
    case["lo"] = max(case["lo"], 0 if op == "prefill" else 1)
    if op == "evict":
        case["keep"] = max(1, int(case["hi"] * rng.choice([0.1, 0.25, 0.5, 0.75])))
        case["recent"] = int(case["keep"] * rng.choice([0.0, 0.1, 0.5]))
    return case


# ---------------------------------------------------------- the 4-bit format
def quantise(x):
    """Codes (c + 8, uint8 [..., D]) and scale bytes (uint8 [..., D / 16]) of fp32 rows.  The quotients are taken in
    64 bits: in 32, a multiplication by a rounded reciprocal takes values next to a border to the wrong side."""
    g = x.float().unflatten(-1, (-1, 16))
    top = g.abs().amax(-1)
    y = top.double() / 7.0
    fraction, e = torch.frexp(y)                                    # y = fraction * 2^e, 1/2 <= fraction < 1
    e = e.clamp(min=-13)
    code = torch.round(torch.ldexp(y, 4 - e)).to(torch.int64) + 8 * (e.to(torch.int64) + 13)
    code = torch.where(torch.isfinite(top), code.clamp(max=225), torch.full_like(code, 255)).to(torch.uint8)
    s = scale_value(code)
    c = torch.where(s[..., None] > 0, g.double() / s[..., None].double(), 0.0)
    c = torch.nan_to_num(torch.round(c), nan=0.0).clamp(-7, 7)
    return (c + 8).to(torch.uint8).flatten(-2), code


def scale_value(code):
    return (code.to(torch.int16) << 7).view(torch.float16).float()


def pack(x, values):
    """Pages [n, H, bs, D] as uint8 pages [n, H, bs, D * 9 / 16]; ``values``: whether they go to the V pool."""
    n, H, bs, D = x.shape
    c, s = quantise(x)
    c = c[..., 0::2] | (c[..., 1::2] << 4)
    if values:
        s = s.transpose(2, 3)
    return torch.cat([c.reshape(n, H, -1), s.reshape(n, H, -1)], 2).reshape(n, H, bs, D * 9 // 16)


def unpack(pages, values):
    """fp32 rows [..., H, bs, D] of uint8 pages [..., H, bs, D * 9 / 16]."""
    bs, D = pages.shape[-2], pages.shape[-1] * 16 // 9
    flat = pages.flatten(-2)
    c, s = flat[..., : bs * D // 2].unflatten(-1, (bs, D // 2)), flat[..., bs * D // 2:]
    x = torch.stack([c & 15, c >> 4], -1).flatten(-2).float().sub_(8.0)
    s = s.unflatten(-1, (D // 16, bs)).transpose(-1, -2) if values else s.unflatten(-1, (bs, D // 16))
    x.unflatten(-1, (-1, 16)).mul_(scale_value(s)[..., None])
    return x


# ------------------------------------------------------------------- prepare
def _lengths(case, seed):
    """Every sequence's length and its number of new tokens: spread evenly over their ranges, in an order of the seed."""
    rs, B, T = np.random.RandomState(seed % (2 ** 31)), case["B"], case.get("T", 1)
    lens = np.rint(np.linspace(case["lo"], case["hi"], B) if B > 1 else [(case["lo"] + case["hi"]) / 2]).astype(np.int64)
    few = max(1, T // 2) if case["op"] == "append" else max(1, T - 7)
    new = few + np.arange(B) * 5 % (T - few + 1)
    order = rs.permutation(B)
    return rs, lens[order], new[order]


def _tables(rs, pages, width, start=0):
    """Random block tables, -1 behind each sequence's pages, over blocks start .. start + sum(pages) - 1."""
    perm, at = rs.permutation(int(sum(pages))) + start, 0
    table = np.full((len(pages), max(1, width)), -1, np.int32)
    for b, n in enumerate(pages):
        table[b, :n] = perm[at: at + n]
        at += n
    return table


def _rows(shape, gen, dtype):
    """Keys, values or queries: unit normal, with every 24th channel or so four times as large."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 1 / 24
    return (x * (1 + 3 * loud)).to(dtype)


def prepare(case, seed):
    rs, lens, new = _lengths(case, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, D, bs, op, dtype = case["B"], case["H"], case["D"], case["bs"], case["op"], DTYPES[case["dtype"]]
    T = case.get("T", 1)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    st = {"case": case}
    if op == "append":
        pages = -(-(lens + new) // bs)
        st.update(starts=dev(lens), new=dev(new))
    else:
        # prefill and weights: lo..hi is the cached prefix, the chunk comes on top (the last row of a ragged chunk is
        # padding in some sequences)
        total = lens + new if op in ("prefill", "weights") else lens
        pages = -(-total // bs)
        st.update(seq_lens=dev(total), cur=dev(new if op in ("prefill", "weights") else np.ones(B)))
    blocks = int(pages.sum())
    extra = int((-(-np.minimum(lens, case["keep"]) // bs)).sum()) if op == "evict" else 0
    st["table"] = dev(_tables(rs, pages, int(pages.max())))
    kv4 = op in ("append", "decode", "prefill") or case.get("cache") == "kv4"
    shape = (blocks + extra, H, bs, D)
    if op == "append":
        # the model's projections, viewed [B, H, T, D]
        for name in ("k_new", "v_new"):
            st[name] = _rows((B, T, H, D), gen, dtype).transpose(1, 2)
        shape = (blocks, H, bs, D * 9 // 16)
        st["k_pool"] = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        st["v_pool"] = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        return st
    for name in ("k_pool", "v_pool"):
        if kv4:
            # in parts: a large cache's fp32 rows need not be held at once
            pool = torch.empty(shape[:3] + (D * 9 // 16,), dtype=torch.uint8, device="cuda")
            part = max(1, (1 << 27) // (H * bs * D))
            loud = 1 + 3 * (torch.rand(D, generator=gen, device="cuda") < 1 / 24)
            for i in range(0, shape[0], part):
                n = min(part, shape[0] - i)
                x = torch.randn((n,) + shape[1:], generator=gen, device="cuda") * loud
                pool[i: i + n] = pack(x.to(dtype).float(), name == "v_pool")
            st[name] = pool
        else:
            st[name] = _rows(shape, gen, dtype)
    if op in ("decode", "prefill", "weights"):
        st["q"] = _rows((B, T, H, D), gen, dtype).transpose(1, 2)
    if op in ("weights", "evict"):
        w = torch.exp(2 * torch.randn(shape[:3], generator=gen, device="cuda"))
        w *= torch.rand(shape[:3], generator=gen, device="cuda") > 0.2  # some keys were never seen
        # the sums of a few earlier queries (a query spreads a weight of one over its keys), or of a long history
        st["weights"] = w / (case["hi"] + T) if op == "weights" else w
        st["weights_out"] = torch.zeros_like(st["weights"])
    if op == "evict":
        st["keep"], st["recent"] = case["keep"], case["recent"]
        st["out_table"] = dev(_tables(rs, -(-np.minimum(lens, case["keep"]) // bs), -(-case["keep"] // bs), blocks))
    return st


# ----------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    return {"append": _append, "decode": _attention, "prefill": _attention, "weights": _weights,
            "evict": _evict}[op](state)


def _run_own(op, st):
    b2pa = _b2pa()
    kp, vp, table = st["k_pool"], st["v_pool"], st["table"]
    if op == "append":
        b2pa.kv4_append(st["k_new"], st["v_new"], kp, vp, table, st["starts"], st["new"])
        return b2pa.kv4_read(kp, vp, table, st["starts"], st["new"], st["k_new"].shape[2], st["k_new"].dtype)
    if op == "decode":
        return b2pa.paged_attention_decode_kv4(st["q"], kp, vp, table, st["seq_lens"], st["cur"])
    if op == "prefill":
        return b2pa.paged_attention_prefill_kv4(st["q"], kp, vp, table, st["seq_lens"], st["cur"])
    if op == "weights":
        return b2pa.accumulate_key_weights(st["q"], kp, st["weights"], table, st["seq_lens"], st["cur"],
                                           window=st["case"]["window"] or None, out=st["weights_out"])
    kept = b2pa.evict_by_weight(kp, vp, st["weights"], table, st["seq_lens"], st["keep"], recent=st["recent"],
                                out_table=st["out_table"])
    return _evicted(st, kept, None if kp.dtype != torch.uint8 else b2pa)


def _evicted(st, kept, b2pa=None):
    """The kept positions, the new pages' weights, and the rows of the new pages (4-bit ones as their values)."""
    kp, vp, keep = st["k_pool"], st["v_pool"], st["keep"]
    if kp.dtype != torch.uint8:
        return {"kept": kept, "weights": st["weights"], "k": kp, "v": vp}
    n = torch.clamp(st["seq_lens"], max=keep)
    if b2pa is not None:
        k, v = b2pa.kv4_read(kp, vp, st["out_table"], torch.zeros_like(n), n, keep, DTYPES[st["case"]["dtype"]])
    else:
        k, v = _read(kp, vp, st["out_table"], torch.zeros_like(n), n, keep, DTYPES[st["case"]["dtype"]])
    return {"kept": kept, "weights": st["weights"], "k": k, "v": v}


def _slots(table, start, length, T, bs):
    """Block and row [B, T] of positions start + t, and which t < length."""
    t = torch.arange(T, device=table.device)
    pos = start.long()[:, None] + t
    live = t < length.long()[:, None]
    page = torch.where(live, pos // bs, torch.zeros_like(pos)).clamp(max=table.shape[1] - 1)
    return table.long().gather(1, page), pos % bs, live


def _read(kp, vp, table, start, length, T, dtype):
    blk, row, live = _slots(table, start, length, T, kp.shape[2])
    blk = blk.clamp(min=0)
    out = []
    for pool, values in ((kp, False), (vp, True)):
        x = unpack(pool, values)[blk, :, row]                       # [B, T, H, D]
        out.append((x * live[:, :, None, None]).transpose(1, 2).to(dtype))
    return tuple(out)


def _append(st):
    kp, vp, table = st["k_pool"], st["v_pool"], st["table"]
    n, H, bs = kp.shape[:3]
    T, D = st["k_new"].shape[2:]
    blk, row, live = _slots(table, st["starts"], st["new"], T, bs)
    blk, row = blk[live], row[live]
    for pool, new, values in ((kp, st["k_new"], False), (vp, st["v_new"], True)):
        c, s = quantise(new.transpose(1, 2)[live].float())          # [tokens, H, D], [tokens, H, D / 16]
        flat = pool.view(n, H, -1)
        codes = flat[..., : bs * D // 2].unflatten(-1, (bs, D // 2))
        codes[blk, :, row] = c[..., 0::2] | (c[..., 1::2] << 4)
        scales = flat[..., bs * D // 2:]
        if values:
            scales.unflatten(-1, (D // 16, bs))[blk, :, :, row] = s
        else:
            scales.unflatten(-1, (bs, D // 16))[blk, :, row] = s
    return _read(kp, vp, table, st["starts"], st["new"], T, st["k_new"].dtype)


def _dense(pool, table, values=False):
    """fp32 rows [B, H, width * bs, D] of the pages of each sequence."""
    pages = pool[table.long().clamp(min=0)]                         # [B, width, H, bs, D or bytes]
    x = unpack(pages, values) if pool.dtype == torch.uint8 else pages.float()
    return x.transpose(1, 2).flatten(2, 3)


def _softmax(st):
    """Weights [B, H, T, L] of every query over the cached keys; zero where a query sees no key."""
    q, table = st["q"].float(), st["table"]
    T, D = q.shape[2:]
    logits = torch.matmul(q, _dense(st["k_pool"], table).transpose(2, 3)) * (1.0 / math.sqrt(D))
    n, cur = st["seq_lens"].long(), st["cur"].long()
    pos = (n - cur)[:, None] + torch.arange(T, device=q.device)
    seen = torch.minimum(n[:, None], pos + 1)
    mask = torch.arange(logits.shape[3], device=q.device) < seen[:, None, :, None]
    logits.masked_fill_(~mask, -math.inf)
    top = logits.amax(3, keepdim=True)
    p = torch.exp(logits.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = p.sum(3, keepdim=True)
    return p.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _attention(st):
    p = _softmax(st)
    v = _dense(st["v_pool"], st["table"], True)
    return torch.matmul(p, v).to(st["q"].dtype)


def _weights(st):
    p = _softmax(st)
    T, window = p.shape[2], st["case"]["window"]
    t, cur = torch.arange(T, device=p.device), st["cur"].long()[:, None]
    counts = (t < cur) & (t >= cur - window) if window else t < cur
    total = (p * counts[:, None, :, None]).sum(2)                   # [B, H, L]
    table, out = st["table"].long(), st["weights_out"]
    bs = out.shape[2]
    total = total.unflatten(2, (-1, bs)).transpose(1, 2)            # [B, pages, H, bs]
    page = torch.arange(table.shape[1], device=p.device) * bs
    n = st["seq_lens"].long()[:, None]
    live = (page[:, None] + torch.arange(bs, device=p.device) < n[:, :, None]) & (table >= 0)[:, :, None]
    used = live.any(2)
    blk = table[used]
    out[blk] = torch.where(live[used][:, None, :], st["weights"][blk] + total[used], out[blk])
    return out


def _evict(st):
    kp, vp, w, table, keep = st["k_pool"], st["v_pool"], st["weights"], st["table"].long(), st["keep"]
    bs, H = w.shape[2], w.shape[1]
    n = st["seq_lens"].long()[:, None]
    k = n.clamp(max=keep)
    dense = w[table.clamp(min=0)].transpose(1, 2).flatten(2, 3)     # [B, H, L]
    j = torch.arange(dense.shape[2], device=w.device)
    recent = min(st["recent"], keep)
    rank = torch.where((j >= n - recent)[:, None], math.inf, dense).masked_fill((j >= n)[:, None], -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices
    if order.shape[2] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[2]), value=dense.shape[2])
    t = torch.arange(keep, device=w.device)
    last = dense.shape[2]
    kept = torch.where((t < k)[:, None], order[..., :keep], last).sort(2).values     # [B, H, keep]
    live = (t < k)[:, None].expand_as(kept)
    src = kept.clamp(max=last - 1)
    head = torch.arange(H, device=w.device)[None, :, None].expand_as(kept)
    s_blk = table[:, None].expand(-1, H, -1).gather(2, src // bs)[live]
    d_blk = st["out_table"].long()[:, None].expand(-1, H, -1).gather(2, (t // bs).expand_as(kept))[live]
    s_row, d_row, h = (src % bs)[live], (t % bs).expand_as(kept)[live], head[live]
    # whole new pages: what is behind the kept rows is zero
    fresh = st["out_table"].long()
    fresh = fresh[fresh >= 0]
    moved = w[s_blk, h, s_row]
    w[fresh] = 0.0
    w[d_blk, h, d_row] = moved
    for pool, values in ((kp, False), (vp, True)):
        if pool.dtype != torch.uint8:
            moved = pool[s_blk, h, s_row]
            pool[fresh] = 0
            pool[d_blk, h, d_row] = moved
            continue
        D = pool.shape[3] * 16 // 9
        flat = pool.view(pool.shape[0], H, -1)
        codes = flat[..., : bs * D // 2].unflatten(-1, (bs, D // 2))
        scales = flat[..., bs * D // 2:]
        scales = (scales.unflatten(-1, (D // 16, bs)).transpose(2, 3) if values
                  else scales.unflatten(-1, (bs, D // 16)))
        c, s = codes[s_blk, h, s_row], scales[s_blk, h, s_row]
        flat[fresh] = 0
        codes[d_blk, h, d_row] = c
        scales[d_blk, h, d_row] = s
    return _evicted(st, torch.where(live, kept, -1).to(torch.int32))


# ---------------------------------------------------------------------- work
def work(case):
    B, H, D, op, es = case["B"], case["H"], case["D"], case["op"], SIZE[case["dtype"]]
    _, lens, new = _lengths(case, 0)
    mean, T = float(lens.mean()), float(new.mean())
    row4 = D * 9 / 16
    if op == "append":
        rows = B * H * T
        # the new rows in, their 4-bit form out, and the values read back from it
        return {"bytes": 2 * rows * (2 * D * es + row4), "flops": 2 * rows * D * 4}
    if op == "evict":
        k = float(np.minimum(lens, case["keep"]).mean())
        row = row4 if case["cache"] == "kv4" else D * es
        values = 2 * D * es + 2 * row if case["cache"] == "kv4" else 0
        return {"bytes": B * H * (4 * mean + k * (4 + 4 + 4 * row + values)), "flops": B * H * mean}
    L = mean + T if op in ("prefill", "weights") else mean
    pairs = B * H * (L if op == "decode" else T * (mean + (T + 1) / 2))
    if op == "weights":
        row = row4 if case["cache"] == "kv4" else D * es
        if case["window"]:
            pairs = B * H * min(T, case["window"]) * (L - (min(T, case["window"]) - 1) / 2)
            T = min(T, case["window"])
        return {"bytes": B * H * (L * (row + 8) + T * D * es), "flops": pairs * 2 * D}
    return {"bytes": B * H * (2 * L * row4 + 2 * T * D * es), "flops": pairs * 4 * D}


# --------------------------------------------------------------------- exact
def _scales64():
    """Every scale the format has, by its byte, in 64 bits."""
    b = np.arange(226)
    e, m = b >> 3, b & 7
    return np.where(e == 0, m / 8.0 * 2.0 ** -14, (1 + m / 8.0) * 2.0 ** (e - 15.0))


def _nearest(x, grid):
    """Index of the nearest grid value, ties to the even index; what is past the grid takes its end."""
    mid = (grid[1:] + grid[:-1]) / 2
    i = torch.bucketize(x, mid)                 # mid[i - 1] < x <= mid[i]
    tie = (i < len(mid)) & (x == mid[i.clamp(max=len(mid) - 1)])
    return torch.where(tie & (i % 2 == 1), i + 1, i)


def _stored64(x):
    """What a row reads back as after 4-bit storage, in 64 bits."""
    grid = torch.from_numpy(_scales64()).to(x.device)
    g = x.double().reshape(x.shape[:-1] + (x.shape[-1] // 16, 16))
    s = grid[_nearest(g.abs().max(dim=-1).values / 7, grid)].unsqueeze(-1)
    code = (g / s.clamp(min=2.0 ** -20)).round().clamp(-7, 7)
    return (code * s).reshape(x.shape)


def _value64(pool, table, n, values):
    """The first n rows [H, n, D] behind one row of the block table, in 64 bits."""
    blocks = table[: -(-n // pool.shape[2])].long()
    if pool.dtype != torch.uint8:
        return pool[blocks].double().permute(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]
    _, H, bs, width = pool.shape
    D = width * 16 // 9
    raw = pool[blocks].permute(1, 0, 2, 3).reshape(H, len(blocks), -1).long()
    byte = raw[:, :, : bs * D // 2].reshape(H, -1, D // 2)
    x = torch.empty(H, byte.shape[1], D, dtype=torch.float64, device=pool.device)
    x[:, :, ::2], x[:, :, 1::2] = (byte % 16 - 8).double(), (byte // 16 - 8).double()
    grid = torch.from_numpy(np.concatenate([_scales64(), np.full(30, np.nan)])).to(pool.device)
    s = grid[raw[:, :, bs * D // 2:]]
    if values:
        s = s.reshape(H, len(blocks), D // 16, bs).permute(0, 1, 3, 2)
    s = s.reshape(H, -1, D // 16)
    return (x * s.repeat_interleave(16, dim=2))[:, :n]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "append":
        t = torch.arange(case["T"], device="cuda")
        live = (t < st["new"][:, None])[:, None, :, None]
        return tuple(torch.where(live, _stored64(st[x]), 0.0) for x in ("k_new", "v_new"))
    if op == "evict":
        return _evict64(st)
    lens, cur = st["seq_lens"].tolist(), st["cur"].tolist()
    q, scale = st["q"].double(), 1 / math.sqrt(case["D"])
    out = st["weights_out"].double() if op == "weights" else torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(lens, cur)):
        K = _value64(st["k_pool"], st["table"][b], n, False)
        first = max(0, m - case["window"]) if op == "weights" and case["window"] else 0
        T = m if op == "weights" else q.shape[2]
        sums = torch.zeros(K.shape[:2], dtype=torch.float64, device="cuda")
        V = _value64(st["v_pool"], st["table"][b], n, True) if op != "weights" else None
        for t0 in range(first, T, 256):
            t1 = min(T, t0 + 256)
            z = q[b, :, t0:t1] @ K.transpose(1, 2) * scale
            last = (n - m + torch.arange(t0, t1, device="cuda")).clamp(max=n - 1)
            hidden = torch.arange(n, device="cuda") > last[:, None]
            p = torch.softmax(z.masked_fill(hidden, -math.inf), dim=2)
            if op == "weights":
                sums += p.sum(1)
            else:
                out[b, :, t0:t1] = p @ V
        if op == "weights":
            bs = out.shape[2]
            for i, blk in enumerate(st["table"][b, : -(-n // bs)].tolist()):
                w = min(bs, n - i * bs)
                out[blk, :, :w] = st["weights"][blk, :, :w].double() + sums[:, i * bs: i * bs + w]
    return out


def _evict64(st):
    """Kept positions, one sequence and head at a time on the host; the rows and weights that move are copies."""
    w, bs, keep = st["weights"].cpu().numpy(), st["weights"].shape[2], st["keep"]
    table, lens = st["table"].cpu().numpy(), st["seq_lens"].tolist()
    kept = np.full((len(lens), w.shape[1], keep), -1, np.int32)
    for b, n in enumerate(lens):
        rows = w[table[b, : -(-n // bs)]].transpose(1, 0, 2).reshape(w.shape[1], -1)[:, :n]
        sure = min(st["recent"], keep, n)
        for h in range(w.shape[1]):
            order = sorted(range(n - sure), key=lambda j: -rows[h, j]) if n > keep else range(n - sure)
            chosen = sorted(list(order)[: min(keep, n) - sure]) + list(range(n - sure, n))
            kept[b, h, : len(chosen)] = chosen
    return {"kept": torch.from_numpy(kept), "weights": None, "k": None, "v": None}
