"""Rules on logits against the header's steps, each rounded to fp32 (numpy): equal."""
import numpy as np
import pytest

import strict_amd
import test_gpu_sample as sampling
from strict_amd import LogitRules
from test_gpu_paged import from16, to16

pytestmark = pytest.mark.gpu


class Rules:
    """Rules as numpy arrays (None: no such rule), by name as LogitRules takes them."""

    def __init__(self, n, **arrays):
        self.n, self.arrays = n, {k: a for k, a in arrays.items() if a is not None}

    def upload(self, ctx, **sizes):
        self.buffers = {k: ctx.upload(a) for k, a in self.arrays.items()}
        a = self.arrays
        numbers = dict(max_tokens=a["tokens"].shape[1] if "tokens" in a else 0,
                       bias_count=len(a["bias_tokens"]) if "bias_tokens" in a else 0,
                       num_masks=len(a["masks"]) if "masks" in a else 0)
        return LogitRules(**self.buffers, **{**numbers, **sizes})

    def free(self):
        for b in self.buffers.values():
            b.free()

    def oracle(self, x):
        a, y = self.arrays, x.astype(np.float32).copy()
        rows, n = y.shape
        one = lambda name, r, other: np.float32(a[name][r]) if name in a else np.float32(other)  # noqa: E731
        with np.errstate(all="ignore"):
            for r in range(rows):
                if "tokens" in a:
                    length = int(np.clip(a["lengths"][r], 0, a["tokens"].shape[1]))
                    prompt = int(np.clip(a["prompts"][r], 0, length)) if "prompts" in a else 0
                    text = a["tokens"][r, :length]
                    behind = text[prompt:]
                    text, behind = (t[(t >= 0) & (t < n)] for t in (text, behind))
                    rep, freq, pres = one("repetition", r, 1), one("frequency", r, 0), one("presence", r, 0)
                    rep = rep if rep > 0 and rep < np.inf else np.float32(1)
                    freq, pres = (v if v == v else np.float32(0) for v in (freq, pres))
                    ids = np.unique(text)
                    v = y[r, ids]
                    y[r, ids] = np.where(v > 0, v / rep, v * rep)
                    ids, times = np.unique(behind, return_counts=True)
                    y[r, ids] = y[r, ids] - (freq * times.astype(np.float32) + pres)
                if "bias_starts" in a:
                    count = len(a["bias_tokens"])
                    lo = int(np.clip(a["bias_starts"][r], 0, count))
                    hi = int(np.clip(a["bias_starts"][r + 1], lo, count))
                    last = {int(a["bias_tokens"][e]): e for e in range(lo, hi)}
                    for t, e in last.items():
                        if 0 <= t < n:
                            y[r, t] += a["bias_values"][e]
                if "masks" in a and 0 <= a["mask_of"][r] < len(a["masks"]):
                    bits = np.unpackbits(np.ascontiguousarray(a["masks"][a["mask_of"][r]]).view(np.uint8), bitorder="little")
                    y[r, bits[:n] == 0] = -np.inf
        return y


def logits(rng, rows, n, dtype):
    """Values and, for the 16-bit types, their patterns."""
    x = rng.normal(0, 3, (rows, n)).astype(np.float32)
    if dtype == "f32":
        return x, x
    bits = to16(x, dtype)
    return from16(bits, dtype).astype(np.float32), bits


def check(ctx, rules, x, bits, dtype="f32", ldx=None, ldy=None, in_place=False):
    rows, n = x.shape
    ldx, ldy = ldx or n, ldy or n
    wide = np.zeros((rows, ldx), bits.dtype)
    wide[:, :n] = bits
    dx = ctx.upload(wide)
    dy = dx if in_place else ctx.upload(np.full((rows, ldy), 7.25, np.float32))
    ctx.adjust_logits(dx, dy, rows, n, rules.upload(ctx), dtype=dtype, ldx=ldx, ldy=ldy)
    ctx.sync()
    got = dy.to_host()
    want = rules.oracle(x)
    same = (got[:, :n] == want) | (np.isnan(got[:, :n]) & np.isnan(want))
    at = np.argwhere(~same)
    assert same.all(), (len(at), at[:5], got[tuple(at[0])], want[tuple(at[0])])
    assert (got[:, n:] == (0 if in_place else 7.25)).all(), "between the rows"
    for b in {id(dx): dx, id(dy): dy}.values():
        b.free()
    rules.free()


def random_rules(rng, rows, n, tokens, biases, masks):
    few = rng.integers(0, n, max(1, n // 10))
    ends = np.concatenate([[0], np.cumsum(rng.integers(0, biases + 1, rows))]).astype(np.int32) if biases else None
    pick = lambda *v: rng.choice(np.float32(v), rows)  # noqa: E731
    return Rules(
        n, tokens=rng.choice(np.concatenate([few, [-1, n, 0, n - 1, np.iinfo(np.int32).max, np.iinfo(np.int32).min]]),
                             (rows, tokens)).astype(np.int32) if tokens else None,
        lengths=rng.integers(0, tokens + 1, rows).astype(np.int32) if tokens else None,
        prompts=rng.integers(-3, tokens + 3, rows).astype(np.int32) if tokens else None,
        repetition=pick(1, 1.3, 0.7, 2), frequency=pick(0, 0.3, -0.1, 1.7), presence=pick(0, 0.6, -0.4),
        bias_starts=ends, bias_tokens=rng.integers(-2, n + 2, max(1, ends[-1])).astype(np.int32) if biases else None,
        bias_values=rng.normal(0, 5, max(1, ends[-1])).astype(np.float32) if biases else None,
        masks=rng.integers(0, 1 << 32, (masks, (n + 31) // 32), dtype=np.uint32) if masks else None,
        mask_of=rng.integers(-1, masks + 1, rows).astype(np.int32) if masks else None)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 5), (2, 33), (5, 2047), (4, 2049), (3, 8191), (2, 50257), (70, 65_537)])
@pytest.mark.parametrize("tokens,biases,masks", [(0, 0, 0), (40, 0, 0), (0, 9, 0), (0, 0, 3), (701, 60, 2)])
def test_rules(ctx, dtype, rows, n, tokens, biases, masks):
    rng = np.random.default_rng(rows + n + tokens)
    x, bits = logits(rng, rows, n, dtype)
    check(ctx, random_rules(rng, rows, n, tokens, biases, masks), x, bits, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,ldx,ldy", [(2048, 2049, 2051), (8193, 8200, 8195), (16_384, 16_385, 16_384)])
def test_strides_and_alignments(ctx, dtype, n, ldx, ldy):
    rng = np.random.default_rng(n)
    x, bits = logits(rng, 7, n, dtype)
    check(ctx, random_rules(rng, 7, n, 100, 20, 2), x, bits, dtype, ldx, ldy)


@pytest.mark.parametrize("n,ld", [(1000, 1000), (2048, 2060), (20_001, 20_003)])
def test_in_place(ctx, n, ld):
    rng = np.random.default_rng(n)
    x, bits = logits(rng, 6, n, "f32")
    check(ctx, random_rules(rng, 6, n, 300, 50, 2), x, bits, ldx=ld, ldy=ld, in_place=True)


def test_long_texts(ctx):
    # one token over and over, more tokens than logits
    rng = np.random.default_rng(1)
    x, bits = logits(rng, 3, 3000, "f32")
    r = random_rules(rng, 3, 3000, 100_001, 0, 0)
    r.arrays["tokens"][1] = 2999
    r.arrays["lengths"][:] = 100_001, 100_000, 99_999
    r.arrays["prompts"][:] = 0, 3, 50_001
    check(ctx, r, x, bits)


def test_values_outside_their_ranges(ctx):
    rng = np.random.default_rng(2)
    rows, n = 12, 5000
    x, bits = logits(rng, rows, n, "f32")
    x[0, :100], x[1, :100], x[2, :100], x[3, :50] = np.inf, -np.inf, np.nan, -0.0
    r = random_rules(rng, rows, n, 60, 12, 2)
    a = r.arrays
    a["lengths"][:4] = np.iinfo(np.int32).max, -1, np.iinfo(np.int32).min, 61
    a["prompts"][:4] = np.iinfo(np.int32).min, 5, 7, np.iinfo(np.int32).max
    a["tokens"][:, :30] = np.arange(30)
    a["repetition"][:] = [0, -1, np.nan, np.inf, -np.inf, 1e-30, 1e30, 2, 1, 1, 1, 1]
    a["frequency"][:] = [1, 1, 1, 1, np.nan, np.inf, -np.inf, np.nan, 3e38, 0, 0, 0]
    a["presence"][:] = [1, 1, 1, 1, 1, np.nan, 1, np.nan, 3e38, np.inf, 0, 0]
    a["bias_starts"][3], a["bias_starts"][5], a["bias_starts"][9] = -7, 1 << 30, 2
    a["bias_values"][:3] = np.inf, -np.inf, np.nan
    a["mask_of"][:4] = np.iinfo(np.int32).min, 2, np.iinfo(np.int32).max, 0
    check(ctx, r, x, bits)


def test_the_same_token_biased_twice(ctx):
    # the last counts; entries of one token far apart, across a row's end
    rng = np.random.default_rng(3)
    x, bits = logits(rng, 2, 9000, "f32")
    tokens = rng.integers(0, 5, 4000).astype(np.int32) * 2000
    r = Rules(9000, bias_starts=np.int32([0, 2500, 4000]), bias_tokens=tokens,
              bias_values=rng.normal(0, 1, 4000).astype(np.float32))
    check(ctx, r, x, bits)


def test_each_rule_alone_and_no_rule(ctx):
    rng = np.random.default_rng(4)
    n, rows = 4100, 4
    full = random_rules(rng, rows, n, 50, 10, 2).arrays
    x, bits = logits(rng, rows, n, "f32")
    text = ("tokens", "lengths")
    bias = ("bias_starts", "bias_tokens", "bias_values")
    for names in ((), text, text + ("repetition",), text + ("frequency", "prompts"), text + ("presence",), bias,
                  ("masks", "mask_of"), ("repetition", "frequency", "presence")):
        check(ctx, Rules(n, **{k: full[k] for k in names}), x, bits)


def test_masks_of_nothing_and_everything(ctx):
    # a row of -infinity throughout samples no token
    rng = np.random.default_rng(5)
    n = 2100
    x, bits = logits(rng, 3, n, "bf16")
    masks = np.zeros((2, (n + 31) // 32), np.uint32)
    masks[1] = 0xffffffff
    r = Rules(n, masks=masks, mask_of=np.int32([0, 1, -1]))
    check(ctx, r, x, bits, "bf16")
    dx, dy, index, work = ctx.upload(bits), ctx.empty((3, n), np.float32), ctx.empty(3, np.int32), ctx.alloc(ctx.sample_workspace(3, n))
    u = ctx.upload(np.float32([0.3, 0.5, 0.9]))
    ctx.adjust_logits(dx, dy, 3, n, r.upload(ctx), dtype="bf16")
    ctx.sample(dy, 3, n, None, None, None, None, u, index, work)
    ctx.sync()
    got = index.to_host()
    assert got[0] == -1 and got[1] >= 0 and got[2] >= 0
    for b in (dx, dy, index, work, u):
        b.free()
    r.free()


def test_adjusted_then_sampled(ctx):
    # what a server does with a step's logits
    rng = np.random.default_rng(6)
    rows, n = 9, 7000
    x, bits = logits(rng, rows, n, "f16")
    r = random_rules(rng, rows, n, 200, 10, 3)
    y = r.oracle(x)
    dx, dy = ctx.upload(bits), ctx.empty((rows, n), np.float32)
    ctx.adjust_logits(dx, dy, rows, n, r.upload(ctx), dtype="f16")
    ctx.sync()
    assert np.array_equal(dy.to_host(), y)
    t, k, p = np.resize(np.float32([0.7, 0, 1.2]), rows), np.resize(np.int32([40, 0]), rows), np.resize(np.float32([1, 0.9]), rows)
    sampling.check(ctx, y, t, k, p, None, rng.random(rows).astype(np.float32))
    dx.free()
    dy.free()
    r.free()


def refused(call, text):
    with pytest.raises(strict_amd.StrictHipError) as e:
        call()
    assert e.value.status == strict_amd.SH_ERR_INVALID_ARGUMENT and text in e.value.message, e.value.message


def test_refusals(ctx):
    rng = np.random.default_rng(7)
    rows, n = 4, 100
    r = random_rules(rng, rows, n, 10, 6, 2)
    whole = r.upload(ctx)
    b = r.buffers
    x, y = ctx.alloc(rows * n * 4), ctx.alloc(rows * n * 4)
    numbers = dict(max_tokens=10, bias_count=whole.struct.bias_count, num_masks=2)
    with_ = lambda **k: LogitRules(**{**b, **numbers, **k})  # noqa: E731
    go = lambda rules=whole, x=x, y=y, rows=rows, n=n, **k: ctx.adjust_logits(x, y, rows, n, rules, **k)  # noqa: E731
    go()
    for bad, text in (((-1, n), "rows"), ((65537, n), "rows"), ((rows, 0), "n must"), ((rows, (1 << 20) + 1), "n must")):
        refused(lambda: go(rows=bad[0], n=bad[1]), text)
    refused(lambda: go(ldx=n - 1), "ld")
    refused(lambda: go(ldy=n - 1), "ldy")
    refused(lambda: go(rows=rows + 1), "x")
    refused(lambda: go(x=None), "x")
    refused(lambda: go(y=x.view(4, x.nbytes - 4), rows=rows - 1), "overlaps x")
    refused(lambda: go(y=x, dtype="f16"), "overlaps x")
    refused(lambda: go(y=x, rows=2, ldx=n, ldy=n + 1), "overlaps x")
    refused(lambda: go(x=x.view(2, x.nbytes - 2), rows=2), "aligned")
    refused(lambda: go(y=y.view(2, y.nbytes - 2), rows=2), "aligned")
    refused(lambda: go(with_(lengths=None)), "lengths")
    refused(lambda: go(with_(max_tokens=-1)), "max_tokens")
    refused(lambda: go(with_(max_tokens=11)), "tokens")
    refused(lambda: go(with_(bias_count=-1)), "bias_count")
    refused(lambda: go(with_(bias_tokens=None)), "bias_tokens")
    refused(lambda: go(with_(bias_values=None)), "bias_values")
    refused(lambda: go(with_(bias_count=numbers["bias_count"] + 1)), "bias_tokens")
    refused(lambda: go(with_(mask_of=None)), "mask_of")
    refused(lambda: go(with_(num_masks=0)), "num_masks")
    refused(lambda: go(with_(num_masks=3)), "masks")
    for name in b:
        size = b[name].nbytes
        area = ctx.alloc(rows * n * 4 + 2 * size)
        for at in (4, size + rows * n * 4 - 4):
            refused(lambda: go(with_(**{name: area.view(at, size)}), y=area.view(size, rows * n * 4)), "overlaps " + name)
        if size > 4:
            refused(lambda: go(with_(**{name: area.view(2, size)})), "4-byte")
        area.free()
    l = strict_amd._lib.load()
    assert l.sh_adjust_logits_f32(ctx.handle, x.ptr, n, y.ptr, n, rows, n, None) == strict_amd.SH_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError):
        go(dtype="f64")
    go(rows=0, x=None, y=None)  # nothing to do
    x.free()
    y.free()
    r.free()
