"""The serving operators over a paged KV cache, as their users call them: sizes,
inputs, one pass, and what that pass computes in 64 bits.

A case is a dict of plain values with an "op":

  norm_rope  the q | k | v rows of a linear: q and k normalised per head and
             rotated, k and v stored in the pages of their positions
  attention  new tokens of a batch of sequences over their pages (one token
             each, or chunks of any length), perhaps within a sliding window
             with the first positions kept visible
  sample     one token per row of logits by temperature, top-k, top-p and
             min-p from given uniform numbers
  copy       pages of every layer's K and V copied within their pools

With `own` false `run` computes a case in elementary torch operations, in 32
bits (the angles and the sampling in 64); with `own` true it calls the
framework on its context's stream and waits for nothing.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ----------------------------------------------------------------

def listed():
    return [
        # a decode step of a small batch: 3 tokens of the Qwen3 shape, launch latency
        {"name": "norm_rope_3", "op": "norm_rope", "dtype": "f16", "batch": 3, "new": 1, "kv": 900,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "theta": 1e6},
        # prompts in chunks: six sequences of up to 2,048 new tokens, far positions
        {"name": "norm_rope_chunks", "op": "norm_rope", "dtype": "bf16", "batch": 6, "new": 2048,
         "kv": 100_003, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "theta": 1e6},
        # one sequence's decode step in one layer of the Qwen3 shape: latency
        {"name": "attn_decode_b1", "op": "attention", "dtype": "f16", "batch": 1, "new": 1,
         "kv": 777, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0,
         "sinks": 0},
        # a serving batch's decode step: 48 sequences of different lengths
        {"name": "attn_decode_b48", "op": "attention", "dtype": "bf16", "batch": 48, "new": 1,
         "kv": 4352, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "sinks": 0},
        # long documents: four sequences of up to 65,537 positions
        {"name": "attn_decode_long", "op": "attention", "dtype": "f16", "batch": 4, "new": 1,
         "kv": 65_537, "heads": 16, "kv_heads": 2, "head_dim": 128, "page": 32, "window": 0,
         "sinks": 0},
        # ragged prompt chunks of the GPT-2 shape
        {"name": "attn_chunks_gpt2", "op": "attention", "dtype": "f16", "batch": 8, "new": 333,
         "kv": 1024, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "window": 0,
         "sinks": 0},
        # a long prompt's chunk of the Qwen3 shape; matrix rate
        {"name": "attn_chunk_8192", "op": "attention", "dtype": "bf16", "batch": 1, "new": 8192,
         "kv": 12_288, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0,
         "sinks": 0},
        # the same with a window: the last 1,024 positions and the first 4
        {"name": "attn_window_1024", "op": "attention", "dtype": "bf16", "batch": 2, "new": 2048,
         "kv": 16_000, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 1024,
         "sinks": 4},
        # one row of GPT-2 logits: latency
        {"name": "sample_1x50257", "op": "sample", "rows": 1, "n": 50257, "ties": False},
        # many rows, logits that came as bf16 (equal values are common): bytes
        {"name": "sample_200x151936", "op": "sample", "rows": 200, "n": 151936, "ties": True},
        # a fork of one sequence: its last page in 12 layers of the GPT-2 shape
        {"name": "copy_fork_gpt2", "op": "copy", "pages": 1, "num_pages": 64, "planes": 24,
         "page_bytes": 16 * 12 * 64 * 2},
        # a compaction: 70 pages in 28 layers of the Qwen3 shape
        {"name": "copy_compact_qwen3", "op": "copy", "pages": 70, "num_pages": 160, "planes": 56,
         "page_bytes": 16 * 8 * 128 * 2},
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
    op = rng.choice(["norm_rope", "attention", "attention", "attention", "sample", "sample", "copy"])
    if op == "norm_rope":
        s = _draw_shape(rng)
        new = _log_int(rng, 1, 2048)
        return {"op": op, "batch": _log_int(rng, 1, max(1, min(64, 8192 // new))), "new": new,
                "kv": new + _log_int(rng, 1, 100_000), "theta": rng.choice([1e4, 1e6]), **s}
    if op == "attention":
        s = _draw_shape(rng)
        if rng.random() < 0.4:
            new, batch = rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 1, 64)
        else:
            new, batch = _log_int(rng, 1, 4096), _log_int(rng, 1, 8)
        # at most the largest listed chunk's scores and the largest listed batch's positions
        longest = min(65_537, int(1.2e9 / (batch * new * s["heads"])),
                      int(1.7e6 / (batch * s["kv_heads"])))
        new = min(new, max(1, longest // 2))
        kv = new + _log_int(rng, 1, max(2, longest - new))
        window = rng.choice([0, 0, 1 + _log_int(rng, 1, 4096)])
        return {"op": op, "batch": batch, "new": new, "kv": kv, "window": window,
                "sinks": rng.choice([0, 4, 100]) if window else 0, **s}
    if op == "sample":
        n = _log_int(rng, 17, 160_000)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(256, 30_000_000 // n))), "n": n,
                "ties": rng.random() < 0.5}
    num = _log_int(rng, 8, 160)
    return {"op": op, "num_pages": num, "pages": _log_int(rng, 1, num // 2), "planes": 2 * rng.randint(1, 28),
            "page_bytes": 16 * _log_int(rng, 8, 4096)}


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


def _visible(n, length, window, sinks):
    """Visible (token, position) pairs of a sequence, and its positions that any token sees."""
    if not window:
        return n * (length - n) + n * (n + 1) // 2, length
    pos = np.arange(length - n, length, dtype=np.int64)
    low = np.maximum(0, pos - window + 1)
    first = max(0, length - n - window + 1)
    return int((pos + 1 - low + np.minimum(sinks, low)).sum()), length - first + min(sinks, first)


def work(case):
    if case["op"] == "copy":
        return {"bytes": 2 * case["pages"] * case["planes"] * case["page_bytes"], "flops": 0}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["n"] * 4 + 5 * 4 + 4), "flops": case["rows"] * case["n"] * 20}
    new, length = _sequences(case)
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        values = sum(new) * (heads + 2 * kv_heads) * d
        return {"bytes": 4 * values + 8 * d, "flops": 10 * values}
    seen = [_visible(n, l, case["window"], case["sinks"]) for n, l in zip(new, length)]
    return {"bytes": 4 * sum(new) * heads * d + 4 * sum(s[1] for s in seen) * kv_heads * d,
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


def _paged(case, g):
    """The pools, a page table of pages in any order, and the batch's lengths. What
    the table holds past a sequence's pages is no page (-1)."""
    new, length = _sequences(case)
    page, d, dtype = case["page"], case["head_dim"], _DTYPES[case["dtype"]]
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
    shape = (num, case["kv_heads"], page, d)
    return {"k": _randn(g, *shape).to(dtype), "v": _randn(g, *shape).to(dtype), "table": table,
            "lengths": _int32(length), "starts": _int32(starts), "tokens": starts[-1],
            "longest_new": max(new), "longest": max(length)}


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] == "copy":
        s["pool"] = torch.randint(-32768, 32767, (case["planes"], case["num_pages"], case["page_bytes"] // 2),
                                  generator=g, device="cuda", dtype=torch.int16)
        order = torch.randperm(case["num_pages"], generator=g, device="cuda").to(torch.int32)
        s["src"], s["dst"] = order[:case["pages"]].clone(), order[case["pages"]:2 * case["pages"]].clone()
        return s
    if case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        # most tokens unlikely, a few dozen well above them
        x = _randn(g, rows, n) * 2.5
        likely = torch.randint(0, n, (rows, 40), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand(rows, 40, generator=g, device="cuda") * 12)
        x[:, n // 3] = -math.inf  # a token that is ruled out
        s["logits"] = x.bfloat16().float() if case["ties"] else x
        pick = lambda values: values[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
        s["temperature"] = pick(torch.tensor([0.0, 0.3, 0.7, 0.7, 1.0, 1.0, 1.5], device="cuda"))
        s["top_k"] = pick(_int32([0, 0, 1, 20, 50, 1000]))
        s["top_p"] = pick(torch.tensor([1.0, 1.0, 0.95, 0.8, 0.3], device="cuda"))
        s["min_p"] = pick(torch.tensor([0.0, 0.0, 0.02, 0.1], device="cuda"))
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["index"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        return s
    s |= _paged(case, g)
    dtype, heads, d = _DTYPES[case["dtype"]], case["heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        s["qkv"] = (_randn(g, s["tokens"], heads + 2 * case["kv_heads"], d) * 1.7).to(dtype)
        s["q_gain"], s["k_gain"] = 1 + 0.2 * _randn(g, d), 1 + 0.2 * _randn(g, d)
        s["q"] = torch.full((s["tokens"], heads, d), 0.5, dtype=dtype, device="cuda")
    else:
        # q and k as head norms leave them; one row behind the last sequence
        s["q"] = (_randn(g, s["tokens"] + 1, heads, d) * 1.5).to(dtype)
        s["out"] = torch.full((s["tokens"] + 1, heads, d), 0.5, dtype=dtype, device="cuda")
    return s


# ---- plain form ---------------------------------------------------------------------

def _token_places(s):
    """Sequence, position and table entry of each token's row."""
    row = torch.arange(s["tokens"], device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = s["lengths"].long()[seq] - starts[seq + 1] + row
    return seq, pos


def _norm_rope_plain(s):
    case = s["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    seq, pos = _token_places(s)
    freq = torch.tensor(case["theta"], dtype=torch.float64) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = pos.double()[:, None, None] * freq.cuda()
    cos, sin = angle.cos().float(), angle.sin().float()
    x = s["qkv"].float()
    x = torch.cat([x[:, :heads], x[:, heads:heads + kv_heads]], 1)
    gain = torch.cat([s["q_gain"].expand(heads, d), s["k_gain"].expand(kv_heads, d)])
    x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-6) * gain
    a, b = x[..., :d // 2], x[..., d // 2:]
    x = torch.cat([a * cos - b * sin, b * cos + a * sin], 2).to(s["qkv"].dtype)
    s["q"].copy_(x[:, :heads])
    at = s["table"].long()[seq, pos // page]
    s["k"][at, :, pos % page] = x[:, heads:]
    s["v"][at, :, pos % page] = s["qkv"][:, heads + kv_heads:]
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _attention_plain(s):
    case = s["case"]
    batch, heads, kv_heads, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    group, n, length = heads // kv_heads, s["longest_new"], s["longest"]
    pages = s["table"].long().clamp_min(0)[:, :-(-length // case["page"])]
    k = s["k"][pages].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, d)[:, :, :length].float()
    v = s["v"][pages].permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, d)[:, :, :length].float()
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
    out = torch.matmul(score.view(batch, kv_heads, group * n, length), v).view(batch, kv_heads, group, n, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, n, heads, d)
    s["out"][row[there]] = out[there].to(s["out"].dtype)
    return s["out"]


def _sample_plain(s):
    n = s["case"]["n"]
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    temperature, p, least, u = (s[name].double()[:, None] for name in ("temperature", "top_p", "min_p", "u"))
    greedy = temperature <= 0
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    w = torch.where(value == top, 1.0, torch.where(greedy, 0.0, torch.exp((value - top) / temperature)))
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k > 0, k, n))
    w = torch.where(torch.arange(n, device="cuda") < k, w, 0.0)
    before = w.cumsum(1) - w
    keep = (before < p * w.sum(1, keepdim=True)) | (p >= 1)
    keep[:, 0] = True
    w = torch.where(keep & (w >= least.clamp_max(1.0)), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.cumsum(1)
    at = (total <= u * total[:, -1:]).sum(1)
    last = n - 1 - (w.flip(1) > 0).int().argmax(1)
    s["index"].copy_(torch.where(top[:, 0] == -math.inf, -1, torch.minimum(at, last)))
    return s["index"]


def _copy_plain(s):
    s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    return s["pool"]


# ---- one pass -----------------------------------------------------------------------

class _Bound:
    """The framework's view of a state: its tensors registered with the context
    and the call on them."""

    context, workspace = None, None

    def __init__(self, s):
        import strict_amd
        if _Bound.context is None:
            _Bound.context = strict_amd.Context(0)
        self.ctx, self.registered = _Bound.context, []
        for t in s.values():
            if isinstance(t, torch.Tensor):
                self.ctx.register_external(t.data_ptr(), t.numel() * t.element_size())
                self.registered.append(t)
        case, p = s["case"], {name: t.data_ptr() for name, t in s.items() if isinstance(t, torch.Tensor)}
        if case["op"] == "copy":
            args = (p["pool"], case["planes"], case["num_pages"], case["page_bytes"], p["src"], p["dst"], case["pages"])
            self.call = lambda: self.ctx.pages_copy(*args)
            return
        if case["op"] == "sample":
            work = self.scratch(self.ctx.sample_workspace(case["rows"], case["n"]))
            args = (p["logits"], case["rows"], case["n"], p["temperature"], p["top_k"], p["top_p"], p["min_p"],
                    p["u"], p["index"], work)
            self.call = lambda: self.ctx.sample(*args)
            return
        kv = strict_amd.PagedKV(p["k"], p["v"], p["table"], p["lengths"], p["starts"], batch=case["batch"],
                                max_pages=s["table"].shape[1], num_pages=s["k"].shape[0], page_size=case["page"],
                                kv_heads=case["kv_heads"], head_dim=case["head_dim"], dtype=case["dtype"])
        if case["op"] == "norm_rope":
            args = (kv, p["qkv"], p["q_gain"], p["k_gain"], p["q"], s["tokens"], case["heads"], 1e-6, case["theta"])
            self.call = lambda: self.ctx.qk_norm_rope_paged(*args)
            return
        tokens = s["tokens"] + 1
        work = self.scratch(self.ctx.attn_paged_workspace(kv, tokens, case["heads"], s["longest_new"]))
        args = (kv, p["q"], p["out"], tokens, case["heads"], s["longest_new"], case["head_dim"] ** -0.5, work)
        self.call = lambda: self.ctx.attn_paged(*args, window=case["window"], sinks=case["sinks"])

    def scratch(self, nbytes):
        """The program's one work buffer, as large as any call has needed."""
        if _Bound.workspace is None or _Bound.workspace.nbytes < nbytes:
            self.ctx.sync()
            if _Bound.workspace is not None:
                _Bound.workspace.free()
            _Bound.workspace = self.ctx.alloc(max(nbytes, 64 << 20))
        return _Bound.workspace

    def __del__(self):
        try:
            self.ctx.sync()
            for t in self.registered:
                self.ctx.unregister_external(t.data_ptr())
        except Exception:
            pass


def run(state):
    op = state["case"]["op"]
    if own:
        if "bound" not in state:
            state["bound"] = _Bound(state)
        state["bound"].call()
        if op == "norm_rope":
            return {"q": state["q"], "k": state["k"], "v": state["v"]}
        return state[{"attention": "out", "sample": "index", "copy": "pool"}[op]]
    return {"norm_rope": _norm_rope_plain, "attention": _attention_plain, "sample": _sample_plain,
            "copy": _copy_plain}[op](state)


# ---- the definition in 64 bits --------------------------------------------------------

def _exact_norm_rope(s):
    case = s["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, length = _sequences(case)
    x = s["qkv"].double()
    k, v, q = s["k"].double(), s["v"].double(), s["q"].double()
    freq = torch.tensor([case["theta"] ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, l) in enumerate(zip(new, length)):
        pos = torch.arange(l - n, l, device="cuda")
        turn = torch.polar(torch.ones(n, 1, d // 2, dtype=torch.float64, device="cuda"), pos[:, None, None] * freq)

        def rotated(y, gain):
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * gain.double()
            z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        rows = x[row:row + n]
        q[row:row + n] = rotated(rows[:, :heads], s["q_gain"])
        at = s["table"][b].long()[pos // page]
        k[at, :, pos % page] = rotated(rows[:, heads:heads + kv_heads], s["k_gain"])
        v[at, :, pos % page] = rows[:, heads + kv_heads:]
        row += n
    return {"q": q, "k": k, "v": v}


def _exact_attention(s):
    case = s["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, length = _sequences(case)
    out = s["out"].double()
    row = 0
    for b, (n, l) in enumerate(zip(new, length)):
        pages = s["table"][b, :-(-l // page)].long()
        pos, p = torch.arange(l - n, l, device="cuda")[:, None], torch.arange(l, device="cuda")
        hidden = p > pos
        if case["window"]:
            hidden |= (p <= pos - case["window"]) & (p >= case["sinks"])
        for h in range(heads):
            kh = s["k"][pages, h * kv_heads // heads].double().reshape(-1, d)[:l]
            vh = s["v"][pages, h * kv_heads // heads].double().reshape(-1, d)[:l]
            score = s["q"][row:row + n, h].double() @ kh.T / math.sqrt(d)
            score[hidden] = -math.inf
            out[row:row + n, h] = torch.softmax(score, -1) @ vh
        row += n
    return out


def _exact_sample(s):
    x = s["logits"].cpu().numpy().astype(np.float64)
    t, k, p, least, u = (s[name].cpu().numpy().astype(np.float64)
                         for name in ("temperature", "top_k", "top_p", "min_p", "u"))
    index = np.zeros(len(x), np.int32)
    for r in range(len(x)):
        order = np.argsort(-x[r], kind="stable")
        kept = order[:1] if t[r] <= 0 else order[:int(k[r])] if k[r] > 0 else order
        w = np.exp((x[r][kept] - x[r][kept[0]]) / (t[r] or 1.0))
        if p[r] < 1:
            at = int(np.searchsorted(np.cumsum(w), p[r] * w.sum(), side="left")) + 1
            kept, w = kept[:at], w[:at]
        kept = np.sort(kept[w >= least[r]])
        w = np.exp((x[r][kept] - x[r][order[0]]) / (t[r] or 1.0))
        c = np.cumsum(w)
        index[r] = kept[min(int(np.searchsorted(c, u[r] * c[-1], side="right")), len(kept) - 1)]
    return torch.from_numpy(index).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            s["pool"][:, b] = s["pool"][:, a]
        return s["pool"]
    return {"norm_rope": _exact_norm_rope, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](s)
