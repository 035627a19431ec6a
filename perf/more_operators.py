"""A decode step in fewer bytes, and rules on its answers: the operators over a paged
cache of 8-bit values, 4-bit weights and adjusted logits, as their users call them:
sizes, inputs, one pass, and what that pass computes in 64 bits.

A case is a dict of plain values with an "op":

  cache8     the q | k | v rows of a linear: q and k normalised per head and rotated,
             k and v quantised into the pages of their positions (E4M3, a power of two
             per row) and the call's rows read back as the values they stand for
  attention8 new tokens of a batch of sequences over such pages, perhaps within a
             sliding window with the first positions kept visible
  gemv4      rows of activations times a matrix of 4-bit weights (E2M1, a power of two
             for 32 of a row)
  logits     penalties for tokens that a row has had, biases and grammar masks on its
             logits

With `own` false `run` computes a case in elementary torch operations, in 32 bits (in 64
what is about to be quantised, and the angles); with `own` true it calls the framework on
its context's stream and waits for nothing.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- the cases ----------------------------------------------------------------

def listed():
    return [
        # a decode step of a small batch: 3 tokens of the Qwen3 shape, launch latency
        {"name": "cache8_3", "op": "cache8", "dtype": "f16", "batch": 3, "new": 1, "kv": 900,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "theta": 1e6},
        # prompts in chunks: six sequences of up to 2,048 new tokens, far positions
        {"name": "cache8_chunks", "op": "cache8", "dtype": "bf16", "batch": 6, "new": 2048,
         "kv": 100_003, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "theta": 1e6},
        # one sequence's decode step in one layer of the Qwen3 shape: latency
        {"name": "attn8_decode_b1", "op": "attention8", "dtype": "f16", "batch": 1, "new": 1,
         "kv": 777, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0,
         "sinks": 0},
        # a serving batch's decode step: 48 sequences of different lengths
        {"name": "attn8_decode_b48", "op": "attention8", "dtype": "bf16", "batch": 48, "new": 1,
         "kv": 8704, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "sinks": 0},
        # long documents: four sequences of up to 131,073 positions
        {"name": "attn8_decode_long", "op": "attention8", "dtype": "f16", "batch": 4, "new": 1,
         "kv": 131_073, "heads": 16, "kv_heads": 2, "head_dim": 128, "page": 32, "window": 0,
         "sinks": 0},
        # ragged prompt chunks of the GPT-2 shape
        {"name": "attn8_chunks_gpt2", "op": "attention8", "dtype": "f16", "batch": 8, "new": 333,
         "kv": 1024, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "window": 0,
         "sinks": 0},
        # a long prompt's chunk of the Qwen3 shape; matrix rate
        {"name": "attn8_chunk_8192", "op": "attention8", "dtype": "bf16", "batch": 1, "new": 8192,
         "kv": 12_288, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "sinks": 0},
        # the attention's output linear of the Qwen3 shape for one token: latency
        {"name": "gemv4_o_b1", "op": "gemv4", "dtype": "f16", "out": "f16", "batch": 1, "k": 2048,
         "n": 1024},
        # the LM head of the Qwen3 shape for one token: bytes
        {"name": "gemv4_head_b1", "op": "gemv4", "dtype": "f16", "out": "f32", "batch": 1, "k": 1024,
         "n": 151_936},
        # a wide layer for a serving batch, sizes that no tile divides
        {"name": "gemv4_wide_b37", "op": "gemv4", "dtype": "bf16", "out": "bf16", "batch": 37,
         "k": 8160, "n": 12_289},
        # one row of GPT-2 logits with a short conversation's penalties: latency
        {"name": "logits_1x50257", "op": "logits", "dtype": "f32", "rows": 1, "n": 50257, "tokens": 600,
         "biases": 20, "masks": 0},
        # a serving batch's logits as a bf16 product leaves them, a third of the rows
        # under a grammar: bytes
        {"name": "logits_200x151936", "op": "logits", "dtype": "bf16", "rows": 200, "n": 151_936,
         "tokens": 4000, "biases": 100, "masks": 7},
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_shape(rng):
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8])
    return {"dtype": rng.choice(["f16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads,
            "head_dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128])}


def draw(rng):
    op = rng.choice(["cache8", "attention8", "attention8", "gemv4", "logits"])
    if op == "cache8":
        s = _draw_shape(rng)
        new = _log_int(rng, 1, 2048)
        return {"op": op, "batch": _log_int(rng, 1, max(1, min(64, 8192 // new))), "new": new,
                "kv": new + _log_int(rng, 1, 100_000), "theta": rng.choice([1e4, 1e6]), **s}
    if op == "attention8":
        s = _draw_shape(rng)
        if rng.random() < 0.4:
            new, batch = rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 1, 64)
        else:
            new, batch = _log_int(rng, 1, 4096), _log_int(rng, 1, 8)
        # at most the largest listed chunk's scores and the largest listed batch's positions
        longest = min(131_073, int(1.2e9 / (batch * new * s["heads"])),
                      int(3.3e6 / (batch * s["kv_heads"])))
        new = min(new, max(1, longest // 2))
        kv = new + _log_int(rng, 1, max(2, longest - new))
        window = rng.choice([0, 0, 1 + _log_int(rng, 1, 4096)])
        return {"op": op, "batch": batch, "new": new, "kv": kv, "window": window,
                "sinks": rng.choice([0, 4, 100]) if window else 0, **s}
    if op == "gemv4":
        k, n = 32 * _log_int(rng, 1, 512), _log_int(rng, 1, 160_000)
        n = min(n, 160_000_000 // k)
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "out": rng.choice(["f32", "16"]),
                "batch": rng.choice([1, 1, _log_int(rng, 1, 64)]), "k": k, "n": n}
    n = _log_int(rng, 17, 160_000)
    return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "n": n,
            "rows": _log_int(rng, 1, max(1, min(256, 30_000_000 // n))),
            "tokens": rng.choice([0, _log_int(rng, 1, 20_000)]),
            "biases": rng.choice([0, _log_int(rng, 1, 300)]), "masks": rng.choice([0, 1, 7])}


def _out_type(case):
    return _DTYPES["f32" if case["out"] == "f32" else case["dtype"]]


def _sequences(case):
    """New tokens and length (new tokens included) of each sequence: the longest
    as the case says, the others below it, the same for every seed."""
    rng = random.Random("%d %d %d" % (case["batch"], case["new"], case["kv"]))
    new, length = [], []
    for b in range(case["batch"]):
        n = case["new"] if b == 0 else rng.randint((case["new"] + 1) // 2, case["new"])
        new.append(n)
        length.append(case["kv"] if b == 0 else n + rng.randint((case["kv"] - n) // 2, case["kv"] - n))
    return new, length


def _row_counts(case):
    """Of each row of logits: its tokens, how many of them are the prompt, its biases and
    its mask (-1: none), the same for every seed."""
    rng = random.Random("%d %d %d" % (case["rows"], case["n"], case["tokens"]))
    rows = []
    for r in range(case["rows"]):
        tokens = case["tokens"] if r == 0 else rng.randint(0, case["tokens"])
        rows.append((tokens, rng.randint(0, tokens), case["biases"] if r == 0 else rng.randint(0, case["biases"]),
                     rng.randrange(case["masks"]) if case["masks"] and rng.random() < 0.33 else -1))
    return rows


def _visible(n, length, window, sinks):
    """Visible (token, position) pairs of a sequence, and its positions that any token sees."""
    if not window:
        return n * (length - n) + n * (n + 1) // 2, length
    pos = np.arange(length - n, length, dtype=np.int64)
    low = np.maximum(0, pos - window + 1)
    first = max(0, length - n - window + 1)
    return int((pos + 1 - low + np.minimum(sinks, low)).sum()), length - first + min(sinks, first)


def work(case):
    if case["op"] == "gemv4":
        n, k, batch = case["n"], case["k"], case["batch"]
        return {"bytes": n * k // 2 + n * k // 32 + batch * k * 2 + batch * n * (4 if case["out"] == "f32" else 2),
                "flops": 2 * batch * n * k}
    if case["op"] == "logits":
        size = 4 if case["dtype"] == "f32" else 2
        rows = _row_counts(case)
        masked = len({r[3] for r in rows if r[3] >= 0})
        return {"bytes": case["rows"] * (case["n"] * (size + 4) + 28) + 4 * sum(r[0] for r in rows)
                + 8 * sum(r[2] for r in rows) + masked * (case["n"] // 8), "flops": 6 * case["rows"] * case["n"]}
    new, length = _sequences(case)
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "cache8":
        # the linear's rows in; q, the pages' rows and what is read of them out
        tokens = sum(new)
        return {"bytes": 2 * tokens * (heads + 2 * kv_heads) * d + 2 * tokens * heads * d
                + 2 * 2 * tokens * kv_heads * (d + 1) + 2 * 2 * tokens * kv_heads * d + 8 * d,
                "flops": 12 * tokens * (heads + 2 * kv_heads) * d}
    seen = [_visible(n, l, case["window"], case["sinks"]) for n, l in zip(new, length)]
    return {"bytes": 4 * sum(new) * heads * d + 2 * sum(s[1] for s in seen) * kv_heads * (d + 1),
            "flops": 4 * heads * d * sum(s[0] for s in seen)}


# ---- what a program has in hand before the call ----------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pow2(e):
    """2^e in 64 bits of whole numbers -1022 .. 1023."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _page_bytes(case):
    return case["kv_heads"] * case["page"] * 2 * (case["head_dim"] + 1)


def _parts(case, pages):
    """A page's K rows and V rows [pages, kv_heads, page, d] and their scales."""
    heads, page, d = case["kv_heads"], case["page"], case["head_dim"]
    rows = heads * page
    values = pages[:, :2 * rows * d].view(-1, 2, heads, page, d)
    scales = pages[:, 2 * rows * d:].view(-1, 2, heads, page)
    return values[:, 0], values[:, 1], scales[:, 0], scales[:, 1]


def _random_rows(g, case, num):
    """Rows of values about as far apart in size as a decoder's, quantised."""
    heads, page, d = case["kv_heads"], case["page"], case["head_dim"]
    x = _randn(g, num, heads, page, d) * torch.exp(0.7 * _randn(g, num, heads, page, 1))
    m, ex = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    q = (x * _pow2(-e).float()).to(torch.float8_e4m3fn).view(torch.uint8)
    return q, (e[..., 0] + 127).to(torch.uint8)


def _paged(case, g):
    """The pages, a table of them in any order, and the batch's lengths. What the table
    holds past a sequence's pages is no page (-1)."""
    new, length = _sequences(case)
    page = case["page"]
    need = [-(-l // page) for l in length]
    num = sum(need) + 3
    order = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    pages = torch.empty(num, _page_bytes(case), dtype=torch.uint8, device="cuda")
    k, v, k_scale, v_scale = _parts(case, pages)
    for i in range(0, num, 4096):  # (a part at a time: the values take eight times the pages' bytes)
        n = min(4096, num - i)
        k[i:i + n], k_scale[i:i + n] = _random_rows(g, case, n)
        v[i:i + n], v_scale[i:i + n] = _random_rows(g, case, n)
    return {"pages": pages, "table": table, "lengths": _int32(length), "starts": _int32(starts),
            "tokens": starts[-1], "longest_new": max(new), "longest": max(length)}


def _prepare_gemv(case, g):
    n, k, dtype = case["n"], case["k"], _DTYPES[case["dtype"]]
    q = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, k // 32, dtype=torch.uint8, device="cuda")
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    for i in range(0, n, 16384):
        w = (_randn(g, min(16384, n - i), k // 32, 32) * 0.02)
        m, ex = torch.frexp(w.abs().amax(-1, keepdim=True))
        e = torch.where(m <= 0.75, ex - 3, ex - 2)
        code = torch.bucketize(w.abs() * _pow2(-e).float(), middle) + torch.where(w < 0, 8, 0)
        code = code.view(len(w), -1)
        q[i:i + len(w)] = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8)
        scales[i:i + len(w)] = (e[..., 0] + 127).to(torch.uint8)
    return {"q": q, "scales": scales, "x": _randn(g, case["batch"], k).to(dtype),
            "y": torch.zeros(case["batch"], n, dtype=_out_type(case), device="cuda")}


def _prepare_logits(case, g):
    rows, n, counts = case["rows"], case["n"], _row_counts(case)
    most = max(1, case["tokens"])
    s = {"x": (_randn(g, rows, n) * 3).to(_DTYPES[case["dtype"]]),
         "y": torch.zeros(rows, n, device="cuda")}
    # few tokens make up most of a text; what lies behind a row's tokens is none
    text = (n * torch.rand(rows, most, generator=g, device="cuda") ** 5).long().clamp_max(n - 1)
    behind = torch.arange(most, device="cuda") >= _int32([c[0] for c in counts])[:, None]
    s["text"] = text.masked_fill(behind, -1).to(torch.int32)
    s["lengths"], s["prompts"] = _int32([c[0] for c in counts]), _int32([c[1] for c in counts])
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
    s["repetition"] = pick([1.0, 1.05, 1.2, 1.7, 0.9])
    s["frequency"], s["presence"] = pick([0.0, 0.1, 0.7, -0.2]), pick([0.0, 0.3, 1.1, -0.5])
    ends = np.cumsum([0] + [c[2] for c in counts])
    s["bias_starts"] = _int32(ends.tolist())
    bias_tokens = [torch.randperm(n, generator=g, device="cuda")[:c[2]] for c in counts] if case["biases"] else []
    # (a row has no more biases than tokens to put them on; what is left over names none)
    s["bias_tokens"] = torch.full((max(1, int(ends[-1])),), -1, dtype=torch.int32, device="cuda")
    for t, at in zip(bias_tokens, ends):
        s["bias_tokens"][int(at):int(at) + len(t)] = t.to(torch.int32)
    s["bias_values"] = _randn(g, max(1, int(ends[-1]))) * 4
    words = (n + 31) // 32
    bits = torch.randint(0, 1 << 32, (max(1, case["masks"]), words), generator=g, device="cuda")
    for _ in range(2):  # an eighth of the tokens are allowed
        bits &= torch.randint(0, 1 << 32, bits.shape, generator=g, device="cuda")
    s["masks"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    s["mask_of"] = _int32([c[3] for c in counts])
    return s


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] in ("gemv4", "logits"):
        s |= (_prepare_gemv if case["op"] == "gemv4" else _prepare_logits)(case, g)
    else:
        s |= _paged(case, g)
        dtype, heads, kv_heads, d = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
        if case["op"] == "cache8":
            s["qkv"] = (_randn(g, s["tokens"], heads + 2 * kv_heads, d) * 1.7).to(dtype)
            s["q_gain"], s["k_gain"] = 1 + 0.2 * _randn(g, d), 1 + 0.2 * _randn(g, d)
            s["q"] = torch.full((s["tokens"], heads, d), 0.5, dtype=dtype, device="cuda")
            s["k"], s["v"] = (torch.full((s["tokens"], kv_heads, d), 0.5, dtype=dtype, device="cuda") for _ in "kv")
        else:
            # q as head norms leave it; one row behind the last sequence
            s["q"] = (_randn(g, s["tokens"] + 1, heads, d) * 1.5).to(dtype)
            s["out"] = torch.full((s["tokens"] + 1, heads, d), 0.5, dtype=dtype, device="cuda")
    if own:
        s["bound"] = _Bound(s)
    return s


# ---- plain form ---------------------------------------------------------------------

def _token_places(s):
    """Sequence, position and table entry of each token's row."""
    row = torch.arange(s["tokens"], device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = s["lengths"].long()[seq] - starts[seq + 1] + row
    return seq, pos


def _quantised(y):
    """Rows of 64-bit values as E4M3 bytes and their scales' bytes."""
    m, ex = torch.frexp(y.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 0.875, ex - 9, ex - 8).clamp_min(-127)
    z = y * _pow2(-e)
    step = _pow2(torch.frexp(z)[1].clamp_min(-5) - 4)  # of E4M3: 2^-3 of a value's power of two, 2^-9 at least
    z = torch.round(z / step) * step
    return z.float().to(torch.float8_e4m3fn).view(torch.uint8), (e[..., 0] + 127).to(torch.uint8)


def _values(q, scale):
    return q.view(torch.float8_e4m3fn).float() * _pow2(scale.long() - 127).float()[..., None]


def _cache8_plain(s):
    case = s["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    seq, pos = _token_places(s)
    freq = torch.tensor(case["theta"], dtype=torch.float64) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = pos.double()[:, None, None] * freq.cuda()

    def rotated(x, gain, cos, sin):
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-6) * gain
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], 2)

    cos, sin = angle.cos(), angle.sin()
    s["q"].copy_(rotated(s["qkv"][:, :heads].float(), s["q_gain"], cos.float(), sin.float()).to(s["q"].dtype))
    k = rotated(s["qkv"][:, heads:heads + kv_heads].double(), s["k_gain"].double(), cos, sin)
    at, row = s["table"].long()[seq, pos // page], pos % page
    kp, vp, ks, vs = _parts(case, s["pages"])
    kp[at, :, row], ks[at, :, row] = _quantised(k)
    vp[at, :, row], vs[at, :, row] = _quantised(s["qkv"][:, heads + kv_heads:].double())
    s["k"].copy_(_values(kp[at, :, row], ks[at, :, row]).to(s["k"].dtype))
    s["v"].copy_(_values(vp[at, :, row], vs[at, :, row]).to(s["v"].dtype))
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _attention8_plain(s):
    case = s["case"]
    batch, heads, kv_heads, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    group, n, length = heads // kv_heads, s["longest_new"], s["longest"]
    pages = s["table"].long().clamp_min(0)[:, :-(-length // case["page"])]
    kp, vp, ks, vs = _parts(case, s["pages"])

    def taken(q, scale):
        x = _values(q[pages], scale[pages]).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, d)
        return x[:, :, :length]

    k, v = taken(kp, ks), taken(vp, vs)
    starts, lengths = s["starts"].long(), s["lengths"].long()
    i = torch.arange(n, device="cuda")
    there = i < (starts[1:] - starts[:-1])[:, None]
    row = (starts[:-1, None] + i).clamp_max(s["tokens"] - 1)
    pos = (lengths - starts[1:] + starts[:-1])[:, None] + i
    p = torch.arange(length, device="cuda")
    seen = p <= pos[..., None]
    if case["window"]:
        seen &= (p > pos[..., None] - case["window"]) | (p < case["sinks"])
    q = s["q"][row].float().view(batch, n, kv_heads, group, d).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * n, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(batch, kv_heads, group, n, length)
    score *= d ** -0.5
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(batch, kv_heads, group * n, length), v.contiguous()).view(batch, kv_heads, group, n, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, n, heads, d)
    s["out"][row[there]] = out[there].to(s["out"].dtype)
    return s["out"]


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _weights(q, scales, dtype):
    value = torch.tensor(_E2M1, dtype=dtype, device="cuda")
    w = torch.stack([value[(q & 15).long()], value[(q >> 4).long()]], -1).view(len(q), -1, 32)
    return (w * _pow2(scales.long() - 127).to(dtype)[..., None]).view(len(q), -1)


def _gemv4_plain(s):
    y = torch.matmul(s["x"].float(), _weights(s["q"], s["scales"], torch.float32).T.contiguous())
    s["y"].copy_(y)
    return s["y"]


def _logits_plain(s):
    rows, n = s["x"].shape
    x = s["x"].float()
    at = torch.arange(s["text"].shape[1], device="cuda")
    there = (at < s["lengths"][:, None]) & (s["text"] >= 0)
    token = s["text"].long().clamp_min(0)
    had = torch.zeros(rows, n, device="cuda").scatter_add_(1, token, there.float()) > 0
    count = torch.zeros(rows, n, device="cuda").scatter_add_(1, token, (there & (at >= s["prompts"][:, None])).float())
    r = s["repetition"][:, None]
    x = torch.where(had, torch.where(x > 0, x / r, x * r), x)
    x = x - (s["frequency"][:, None] * count + torch.where(count > 0, s["presence"][:, None], 0.0))
    entry = torch.arange(len(s["bias_tokens"]), device="cuda")
    row = torch.searchsorted(s["bias_starts"].long(), entry, right=True) - 1
    named = (row < rows) & (s["bias_tokens"] >= 0)
    row, name = row[named], s["bias_tokens"].long()[named]
    x[row, name] = x[row, name] + s["bias_values"][named]
    token = torch.arange(n, device="cuda")
    bits = (s["masks"][s["mask_of"].long().clamp_min(0)][:, token // 32] >> (token % 32).to(torch.int32)) & 1
    s["y"].copy_(torch.where((bits != 0) | (s["mask_of"] < 0)[:, None], x, -math.inf))
    return s["y"]


# ---- one pass -----------------------------------------------------------------------

class _Bound:
    """The framework's view of a state: its tensors registered with the context
    and the calls on them."""

    context, workspace = None, None

    def __init__(self, s):
        import strict_amd
        if _Bound.context is None:
            _Bound.context = strict_amd.Context(0)
        ctx = self.ctx = _Bound.context
        self.registered = []
        for t in s.values():
            if isinstance(t, torch.Tensor):
                ctx.register_external(t.data_ptr(), t.numel() * t.element_size())
                self.registered.append(t)
        torch.cuda.synchronize()  # the inputs were made on another stream
        case, p = s["case"], {name: t.data_ptr() for name, t in s.items() if isinstance(t, torch.Tensor)}
        if case["op"] == "gemv4":
            batch, k, n, dtype = case["batch"], case["k"], case["n"], case["dtype"]
            weights = self.weights = ctx.alloc(ctx.e2m1_tiles_bytes(n, k))  # laid out once
            ctx.pack_e2m1_tiles(p["q"], p["scales"], weights, n, k)
            out = "f32" if case["out"] == "f32" else dtype
            self.call = lambda: ctx.gemv_w4a16(p["x"], weights, p["y"], batch, k, n, dtype=dtype, out=out)
            return
        if case["op"] == "logits":
            rules = strict_amd.LogitRules(
                tokens=p["text"], max_tokens=s["text"].shape[1], lengths=p["lengths"], prompts=p["prompts"],
                repetition=p["repetition"], frequency=p["frequency"], presence=p["presence"],
                bias_starts=p["bias_starts"], bias_tokens=p["bias_tokens"], bias_values=p["bias_values"],
                bias_count=len(s["bias_tokens"]), masks=p["masks"], mask_of=p["mask_of"], num_masks=len(s["masks"]))
            self.call = lambda: ctx.adjust_logits(p["x"], p["y"], case["rows"], case["n"], rules, dtype=case["dtype"])
            return
        kv = strict_amd.PagedKV8(p["pages"], p["table"], p["lengths"], p["starts"], batch=case["batch"],
                                 max_pages=s["table"].shape[1], num_pages=len(s["pages"]), page_size=case["page"],
                                 kv_heads=case["kv_heads"], head_dim=case["head_dim"], dtype=case["dtype"])
        if case["op"] == "cache8":
            tokens, args = s["tokens"], (case["heads"], 1e-6, case["theta"])

            def store_and_read():
                ctx.qk_norm_rope_paged(kv, p["qkv"], p["q_gain"], p["k_gain"], p["q"], tokens, *args)
                ctx.paged_read(kv, p["k"], p["v"], tokens)
            self.call = store_and_read
            return
        tokens = s["tokens"] + 1
        work = self.scratch(ctx.attn_paged_workspace(kv, tokens, case["heads"], s["longest_new"]))
        args = (kv, p["q"], p["out"], tokens, case["heads"], s["longest_new"], case["head_dim"] ** -0.5, work)
        self.call = lambda: ctx.attn_paged(*args, window=case["window"], sinks=case["sinks"])

    def scratch(self, nbytes):
        """The program's one work buffer, as large as any call needs."""
        if _Bound.workspace is None:
            _Bound.workspace = self.ctx.alloc(256 << 20)
        if _Bound.workspace.nbytes < nbytes:
            raise RuntimeError("a work buffer of %d bytes" % nbytes)
        return _Bound.workspace

    def __del__(self):
        try:
            self.ctx.sync()
            for t in self.registered:
                self.ctx.unregister_external(t.data_ptr())
            if hasattr(self, "weights"):
                self.weights.free()
        except Exception:
            pass


def run(state):
    op = state["case"]["op"]
    if own:
        state["bound"].call()
        if op == "cache8":
            return {"q": state["q"], "k": state["k"], "v": state["v"]}
        return state["out" if op == "attention8" else "y"]
    return {"cache8": _cache8_plain, "attention8": _attention8_plain, "gemv4": _gemv4_plain,
            "logits": _logits_plain}[op](state)


# ---- the definition in 64 bits --------------------------------------------------------

def _e4m3_table():
    """The values of the bytes 0 .. 126, from their exponents and fractions."""
    return torch.tensor([(b & 7) * 2.0 ** -9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10) for b in range(127)],
                        dtype=torch.float64, device="cuda")


def _nearest(x):
    """Rows as the values that their E4M3 bytes and scales stand for: the nearest of the
    table's, of two as near the even byte."""
    table = _e4m3_table()
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448.0))
    z = x.abs() / torch.exp2(e)
    high = torch.searchsorted(table, z.contiguous()).clamp(1, 126)
    below, above = z - table[high - 1], table[high] - z
    byte = torch.where((above < below) | ((above == below) & (high % 2 == 0)), high, high - 1)
    return torch.where(x < 0, -1.0, 1.0) * table[byte] * torch.exp2(e)


def _exact_cache8(s):
    case = s["case"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    new, length = _sequences(case)
    x = s["qkv"].double()
    freq = torch.tensor([case["theta"] ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
    pos = torch.cat([torch.arange(l - n, l, device="cuda") for n, l in zip(new, length)])
    turn = torch.polar(torch.ones(len(pos), 1, d // 2, dtype=torch.float64, device="cuda"), pos[:, None, None] * freq)

    def rotated(y, gain):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * gain.double()
        z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    return {"q": rotated(x[:, :heads], s["q_gain"]),
            "k": _nearest(rotated(x[:, heads:heads + kv_heads], s["k_gain"])),
            "v": _nearest(x[:, heads + kv_heads:])}


def _exact_attention8(s):
    case = s["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, length = _sequences(case)
    out = s["out"].double()
    table = _e4m3_table()
    nan = torch.full((1,), math.nan, dtype=torch.float64, device="cuda")
    table = torch.cat([table, nan, -table, nan])
    rows = kv_heads * page
    row = 0
    for b, (n, l) in enumerate(zip(new, length)):
        held = s["pages"][s["table"][b, :-(-l // page)].long()]
        pos, p = torch.arange(l - n, l, device="cuda")[:, None], torch.arange(l, device="cuda")
        hidden = p > pos
        if case["window"]:
            hidden |= (p <= pos - case["window"]) & (p >= case["sinks"])

        def head_of(which, h):
            first = which * rows * d + h * page * d
            scale = 2 * rows * d + which * rows + h * page
            x = table[held[:, first:first + page * d].reshape(-1, d)[:l].long()]
            return x * torch.exp2(held[:, scale:scale + page].reshape(-1)[:l].double() - 127)[:, None]

        for kh in range(kv_heads):
            k, v = head_of(0, kh), head_of(1, kh)
            for h in range(kh * heads // kv_heads, (kh + 1) * heads // kv_heads):
                score = s["q"][row:row + n, h].double() @ k.T / math.sqrt(d)
                score[hidden] = -math.inf
                out[row:row + n, h] = torch.softmax(score, -1) @ v
        row += n
    return out


def _exact_gemv4(s):
    case = s["case"]
    y = torch.zeros(case["batch"], case["n"], dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for i in range(0, case["n"], 8192):
        q, scale = s["q"][i:i + 8192].int(), s["scales"][i:i + 8192].double()
        for nibble in (0, 1):  # even places of a row, then odd ones
            code = (q >> (4 * nibble)) & 15
            e, f = (code >> 1) & 3, (code & 1).double()
            w = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2(e.double() - 1))
            w = torch.where(code >= 8, -w, w) * torch.exp2(scale - 127).repeat_interleave(16, 1)
            y[:, i:i + 8192] += x[:, nibble::2].contiguous() @ w.T.contiguous()
    return y


def _exact_logits(s):
    x = s["x"].double().cpu().numpy()
    h = {name: t.cpu().numpy() for name, t in s.items() if isinstance(t, torch.Tensor) and name not in ("x", "y")}
    rows, n = x.shape
    for r in range(rows):
        text = h["text"][r, :h["lengths"][r]]
        ids = np.unique(text)
        v = x[r, ids]
        x[r, ids] = np.where(v > 0, v / np.float64(h["repetition"][r]), v * np.float64(h["repetition"][r]))
        ids, times = np.unique(text[h["prompts"][r]:], return_counts=True)
        x[r, ids] -= np.float64(h["frequency"][r]) * times + np.float64(h["presence"][r])
        for e in range(h["bias_starts"][r], h["bias_starts"][r + 1]):
            if h["bias_tokens"][e] >= 0:
                x[r, h["bias_tokens"][e]] += np.float64(h["bias_values"][e])
        if h["mask_of"][r] >= 0:
            words = np.ascontiguousarray(h["masks"][h["mask_of"][r]]).view(np.uint8)
            x[r, np.unpackbits(words, bitorder="little")[:n] == 0] = -np.inf
    return torch.from_numpy(x).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    return {"cache8": _exact_cache8, "attention8": _exact_attention8, "gemv4": _exact_gemv4,
            "logits": _exact_logits}[case["op"]](s)
