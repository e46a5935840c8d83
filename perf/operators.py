"""Cases and plain forms of the 8-bit KV cache operators and of the token log probabilities.

Four operators: the append of new tokens to an 8-bit paged cache, decode and varlen prefill
attention over it, and the log probabilities, entropy and top alternatives of logits rows. Each
is written here once more in elementary torch operations (``own`` false), and called as a user's
program calls it (``own`` true).

The cache holds bytes (e4m3 or int8) of shape [num_blocks, kv_heads, 16, d] and one f32 scale for
each (block, head) of K and of V: a value is its byte times the scale. Scales written by the
append are powers of two, so that a quotient x / scale is exact and rounds once.
"""

import math

import numpy as np
import torch

own = False

BS = 16  # tokens per block
QMAX = {"e4m3": 448.0, "i8": 127.0}
BYTES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
FLOATS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ---- cases ----------------------------------------------------------------------------------

def listed():
    return [
        # One decode step of 64 running sequences: each appends its new token (latency).
        {"name": "append step, 64 sequences", "op": "append", "heads": 32, "kv_heads": 8, "d": 128,
         "fmt": "e4m3", "dtype": "bf16", "seqs": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 512,
         "ctx_hi": 4096, "lens": 1},
        # A batch of prompts behind cached prefixes of odd lengths (ragged blocks at both ends).
        {"name": "append prompts", "op": "append", "heads": 28, "kv_heads": 4, "d": 128, "fmt": "i8",
         "dtype": "f16", "seqs": 16, "new_lo": 100, "new_hi": 1990, "ctx_lo": 128, "ctx_hi": 2048,
         "lens": 2},
        # Long documents read into the cache at once.
        {"name": "append long documents", "op": "append", "heads": 32, "kv_heads": 8, "d": 128,
         "fmt": "e4m3", "dtype": "bf16", "seqs": 8, "new_lo": 5000, "new_hi": 8192, "ctx_lo": 5000,
         "ctx_hi": 8192, "lens": 3},
        # One chat with a small model, a short context (latency).
        {"name": "decode one sequence", "op": "decode", "heads": 14, "kv_heads": 2, "d": 64,
         "fmt": "i8", "dtype": "bf16", "seqs": 1, "ctx_lo": 511, "ctx_hi": 511, "lens": 4},
        # A serving batch, contexts U[512, 4096].
        {"name": "decode batch 64", "op": "decode", "heads": 32, "kv_heads": 8, "d": 128,
         "fmt": "e4m3", "dtype": "bf16", "seqs": 64, "ctx_lo": 512, "ctx_hi": 4096, "lens": 5},
        # Seven query heads to a KV head, f16 model, a ragged batch from one token on.
        {"name": "decode ragged n_rep 7", "op": "decode", "heads": 28, "kv_heads": 4, "d": 128,
         "fmt": "i8", "dtype": "f16", "seqs": 59, "ctx_lo": 1, "ctx_hi": 6438, "lens": 6},
        # Long contexts, U[16384, 32768].
        {"name": "decode long contexts", "op": "decode", "heads": 32, "kv_heads": 8, "d": 128,
         "fmt": "e4m3", "dtype": "bf16", "seqs": 16, "ctx_lo": 16384, "ctx_hi": 32768, "lens": 7},
        # Prompts behind cached prefixes.
        {"name": "prefill prompts", "op": "prefill", "heads": 32, "kv_heads": 8, "d": 128,
         "fmt": "e4m3", "dtype": "bf16", "seqs": 16, "new_lo": 100, "new_hi": 2048, "ctx_lo": 128,
         "ctx_hi": 2048, "lens": 8},
        # The last chunk of a long document: few queries over much cache.
        {"name": "prefill chunk of a document", "op": "prefill", "heads": 28, "kv_heads": 4, "d": 128,
         "fmt": "i8", "dtype": "bf16", "seqs": 1, "new_lo": 509, "new_hi": 509, "ctx_lo": 30001,
         "ctx_hi": 30001, "lens": 9},
        # The answer of one chat: one row, 20 alternatives (latency).
        {"name": "logprobs one row", "op": "logprobs", "dtype": "f32", "rows": 1, "vocab": 151936,
         "pad": 0, "top_k": 20, "masked": False},
        # The answers of a serving batch, some under a grammar that allows few tokens.
        {"name": "logprobs batch 64", "op": "logprobs", "dtype": "f32", "rows": 64, "vocab": 128256,
         "pad": 0, "top_k": 20, "masked": True},
        # Scoring given documents: every position of a prompt, bf16 logits, 5 alternatives.
        {"name": "logprobs of a document", "op": "logprobs", "dtype": "bf16", "rows": 2048,
         "vocab": 151643, "pad": 293, "top_k": 5, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 152000)
        rows = _log_int(rng, 1, max(1, min(4096, 150_000_000 // vocab)))
        return {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "rows": rows, "vocab": vocab,
                "pad": rng.choice([0, 0, 1, 37]), "top_k": rng.choice([0, 1, 5, 20]),
                "masked": rng.random() < 0.5}
    heads, kv_heads, d = rng.choice([(32, 8, 128), (28, 4, 128), (14, 2, 64)] if op != "prefill"
                                    else [(32, 8, 128), (28, 4, 128)])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "d": d,
            "fmt": rng.choice(["e4m3", "i8"]), "dtype": rng.choice(["bf16", "f16"])}
    lens = rng.randrange(1 << 20)
    if op == "append":
        hi = _log_int(rng, 1, 8192)
        seqs = _log_int(rng, 1, max(1, min(256, 50_000 // hi)))
        ctx = max(hi, _log_int(rng, 16, 8192))
        return dict(case, seqs=seqs, new_lo=max(1, hi // 3), new_hi=hi, ctx_lo=max(1, ctx // 3),
                    ctx_hi=ctx, lens=lens)
    if op == "decode":
        hi = _log_int(rng, 16, 32768)
        seqs = _log_int(rng, 1, max(1, min(256, 300_000 // hi)))
        return dict(case, seqs=seqs, ctx_lo=max(1, hi // rng.choice([1, 2, 8])), ctx_hi=hi, lens=lens)
    new = _log_int(rng, 128, 2048)
    ctx = max(new, _log_int(rng, 128, min(8192, 12_000_000 // new)))
    seqs = max(1, min(16, 12_000_000 // (new * ctx)))
    return dict(case, seqs=seqs, new_lo=max(1, new // 4), new_hi=new, ctx_lo=max(1, ctx // 4),
                ctx_hi=ctx, lens=lens)


def _lengths(case):
    """Context lengths and new-token counts, by the case alone."""
    rng = np.random.default_rng(case["lens"])
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["seqs"])
    new = np.ones_like(ctx)
    if "new_lo" in case:
        new = rng.integers(case["new_lo"], case["new_hi"] + 1, size=case["seqs"])
    ctx[0] = case["ctx_hi"]
    return ctx, np.minimum(new, ctx)


# ---- inputs ---------------------------------------------------------------------------------

def _pow2_scale(a, fmt):
    """The smallest power of two s >= 2^-126 with a <= qmax * s (a: f32, >= 0)."""
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1)
    top, bits = (0.875, 9) if fmt == "e4m3" else (127.0 / 128.0, 7)  # qmax = top * 2^bits
    e = torch.where(m > top, e - bits + 1, e - bits)
    e = torch.where(a > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(a), e)


def _to_bytes(x, fmt):
    """f32 values already divided by their scale -> 8 bits, nearest, ties to even."""
    if fmt == "e4m3":
        return x.to(torch.float8_e4m3fn)
    return torch.round(x).clamp(-127, 127).to(torch.int8)


def _raw(t):
    return t.view(torch.uint8)


def _pool(case, gen, blocks, stale):
    """A filled pool: keys with louder channels, values of another loudness for each head."""
    H, d, fmt = case["kv_heads"], case["d"], case["fmt"]
    out = []
    for kind in ("k", "v"):
        loud = torch.randn((1, H, 1, d if kind == "k" else 1), device=DEV, generator=gen).mul_(0.5).exp_()
        bytes_ = torch.empty((blocks, H, BS, d), dtype=BYTES[fmt], device=DEV)
        scale = torch.empty((blocks, H), dtype=torch.float32, device=DEV)
        for b0 in range(0, blocks, 8192):
            n = min(8192, blocks - b0)
            x = torch.randn((n, H, BS, d), device=DEV, generator=gen).mul_(loud)
            s = _pow2_scale(x.abs().amax((2, 3)), fmt)
            bytes_[b0:b0 + n] = _to_bytes(x / s[:, :, None, None], fmt)
            scale[b0:b0 + n] = s
        out += [bytes_, scale]
    kc, ks, vc, vs = out
    if stale is not None:  # what an earlier owner left behind the last token, NaN bytes among it
        ids, first = stale
        rows = torch.arange(BS, device=DEV)[None, :] >= first[:, None]
        for c in (kc, vc):
            raw = _raw(c)[ids]
            junk = torch.randint(0, 256, raw.shape, device=DEV, generator=gen, dtype=torch.uint8)
            _raw(c)[ids] = torch.where(rows[:, None, :, None], junk, raw)
    return kc, ks, vc, vs


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        full = torch.empty((R, V + case["pad"]), dtype=FLOATS[case["dtype"]], device=DEV)
        for r0 in range(0, R, 256):
            n = min(256, R - r0)
            x = torch.randn((n, V + case["pad"]), device=DEV, generator=gen).mul_(2.0)
            peaks = torch.randint(0, V, (n, 8), device=DEV, generator=gen)
            x.scatter_add_(1, peaks, torch.rand((n, 8), device=DEV, generator=gen).mul_(12.0))
            full[r0:r0 + n] = x.to(full.dtype)
        ids = torch.randint(0, V, (R,), device=DEV, generator=gen, dtype=torch.int32)
        if case["masked"]:  # every third row allows about seven tokens, the given one among them
            keep = torch.rand((R, V + case["pad"]), device=DEV, generator=gen) < 7.0 / V
            keep |= (torch.arange(R, device=DEV) % 3 != 0)[:, None]
            keep.scatter_(1, ids.long()[:, None], True)
            full.masked_fill_(~keep, -math.inf)
        return {"op": "logprobs", "logits": full[:, :V], "ids": ids, "top_k": case["top_k"]}
    ctx, new = _lengths(case)
    pages = (ctx + BS - 1) // BS
    total = int(pages.sum())
    blocks = total + 7
    perm = torch.randperm(blocks, device=DEV, generator=gen).to(torch.int32)
    tables = torch.zeros((len(ctx), int(pages.max())), dtype=torch.int32, device=DEV)
    row = torch.from_numpy(np.repeat(np.arange(len(ctx)), pages)).to(DEV)
    col = torch.from_numpy(np.concatenate([np.arange(n) for n in pages])).to(DEV)
    tables[row, col] = perm[:total]
    ctx_dev = torch.from_numpy(ctx.astype(np.int32)).to(DEV)
    state = {"op": case["op"], "fmt": case["fmt"], "tables": tables, "ctx": ctx_dev,
             "max_ctx": int(ctx.max()), "n_rep": case["heads"] // case["kv_heads"],
             "scale": 1.0 / math.sqrt(case["d"]), "total_blocks": total}
    stale = None
    if case["op"] != "append":
        last = tables[torch.arange(len(ctx), device=DEV), torch.from_numpy(pages - 1).to(DEV)].long()
        stale = (last, torch.from_numpy((ctx - 1) % BS + 1).to(DEV))
    state["kc"], state["ks"], state["vc"], state["vs"] = _pool(case, gen, blocks, stale)
    dt = FLOATS[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, device=DEV, generator=gen).to(dt)

    cu = np.concatenate([[0], np.cumsum(new)])
    state["cu"] = torch.from_numpy(cu.astype(np.int32)).to(DEV)
    state["max_new"], state["total_new"] = int(new.max()), int(cu[-1])
    if case["op"] == "append":
        loud = torch.randn((1, case["kv_heads"], case["d"]), device=DEV, generator=gen).mul_(0.7).exp_()
        state["key"] = (rand(int(cu[-1]), case["kv_heads"], case["d"]).float() * loud).to(dt)
        state["value"] = rand(int(cu[-1]), case["kv_heads"], case["d"])
    else:
        state["q"] = rand(int(cu[-1]), case["heads"], case["d"])
    return state


# ---- one pass -------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "decode": _decode, "prefill": _prefill,
            "logprobs": _logprobs}[state["op"]](state)


def _run_own(s):
    from flour_b200 import ops
    if s["op"] == "logprobs":
        return ops.token_logprobs(s["logits"], s["ids"], s["top_k"])
    pool = (s["kc"], s["vc"], s["ks"], s["vs"])
    if s["op"] == "append":
        cu = s["cu"] if s["max_new"] > 1 else None
        ops.paged_append_kv8(*pool, s["key"], s["value"], s["tables"], s["ctx"], cu)
        return pool
    if "ws" not in s:  # the workspace that a program keeps
        s["ws"] = ops.Workspace()
    if s["op"] == "decode":
        return ops.paged_decode_kv8(s["q"], *pool, s["tables"], s["ctx"], s["n_rep"], s["scale"],
                                    s["max_ctx"], s["ws"])
    return ops.paged_prefill_kv8(s["q"], *pool, s["cu"], s["ctx"], s["tables"], s["n_rep"],
                                 s["scale"], s["max_new"], s["max_ctx"], s["total_blocks"], s["ws"])


def _append(s):
    """Each sequence's touched blocks at once: [sequences, touched blocks, ...]. Columns past a
    sequence's last block repeat it, and write what it gets once more."""
    fmt, ctx, cu = s["fmt"], s["ctx"].long(), s["cu"].long()
    start = ctx - (cu[1:] - cu[:-1])
    first, last = start // BS, (ctx - 1) // BS
    width = (s["max_new"] + BS - 2) // BS + 1
    logical = torch.minimum(first[:, None] + torch.arange(width, device=DEV), last[:, None])
    ids = s["tables"].long().gather(1, logical)
    pos = logical[:, :, None] * BS + torch.arange(BS, device=DEV)
    fresh = (pos >= start[:, None, None]) & (pos < ctx[:, None, None])       # new rows
    kept = pos < start[:, None, None]                                        # rows held before
    tok = (cu[:-1, None, None] + pos - start[:, None, None]).clamp(0, s["total_new"] - 1)
    held = (logical * BS < start[:, None])[:, :, None]
    fresh, kept = fresh[:, :, None, :, None], kept[:, :, None, :, None]
    for cache, scale, x in ((s["kc"], s["ks"], s["key"]), (s["vc"], s["vs"], s["value"])):
        x = x[tok].float().permute(0, 1, 3, 2, 4)                            # [.., head, row, d]
        need = _pow2_scale(torch.where(fresh, x, 0.0).abs().amax((3, 4)), fmt)
        before = scale[ids]
        after = torch.where(held, torch.maximum(before, need), need)
        old = _raw(cache)[ids].view(cache.dtype)
        moved = _to_bytes(old.float() * (before / after)[..., None, None], fmt)
        put = _to_bytes(torch.where(fresh, x / after[..., None, None], 0.0), fmt)
        _raw(cache)[ids] = torch.where(fresh, _raw(put), torch.where(kept, _raw(moved), _raw(old)))
        scale[ids] = after
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _gathered(s, cache, scale):
    """[sequences, kv heads, positions, d] in f32, dead positions zero."""
    ids = s["tables"].long()
    x = _raw(cache)[ids].view(cache.dtype).float() * scale[ids][..., None, None]
    S, nb, H, _, d = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(S, H, nb * BS, d)
    live = torch.arange(nb * BS, device=DEV)[None, :] < s["ctx"][:, None]
    return torch.where(live[:, None, :, None], x, 0.0)


def _attend(s, q, limit):
    """q [sequences, kv heads, rows, d]; row r sees positions <= limit [sequences, rows]."""
    k, v = _gathered(s, s["kc"], s["ks"]), _gathered(s, s["vc"], s["vs"])
    score = (q @ k.transpose(2, 3)) * s["scale"]
    hidden = torch.arange(k.shape[2], device=DEV)[None, None, :] > limit[:, :, None]
    score = score.masked_fill_(hidden[:, None], -math.inf)
    e = (score - score.amax(3, keepdim=True)).exp_()
    return (e @ v) / e.sum(3, keepdim=True)


def _decode(s):
    q = s["q"]
    S, heads, d = q.shape
    r = s["n_rep"]
    limit = (s["ctx"].long() - 1)[:, None].expand(S, r)
    return _attend(s, q.float().reshape(S, heads // r, r, d), limit).reshape(S, heads, d).to(q.dtype)


def _prefill(s):
    q, cu, r, n = s["q"], s["cu"].long(), s["n_rep"], s["max_new"]
    T, heads, d = q.shape
    S = cu.numel() - 1
    new = cu[1:] - cu[:-1]
    i = torch.arange(n, device=DEV)
    tok = (cu[:-1, None] + i).clamp(max=T - 1)                                # padded rows repeat a token
    x = q[tok].float().reshape(S, n, heads // r, r, d).permute(0, 2, 1, 3, 4).reshape(S, heads // r, n * r, d)
    limit = ((s["ctx"].long() - new)[:, None] + i).clamp(max=s["max_ctx"] - 1).repeat_interleave(r, 1)
    o = _attend(s, x, limit).reshape(S, heads // r, n, r, d).permute(0, 2, 1, 3, 4).reshape(S, n, heads, d)
    seq = torch.searchsorted(cu, torch.arange(T, device=DEV), right=True) - 1
    return o[seq, torch.arange(T, device=DEV) - cu[seq]].to(q.dtype)


def _logprobs(s):
    x = s["logits"].float()
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1)
    log_z = z.log()
    given = d.gather(1, s["ids"].long()[:, None])[:, 0] - log_z
    entropy = log_z - torch.where(e > 0, e * d, 0.0).sum(1) / z
    k = s["top_k"]
    top, ids = torch.sort(d, dim=1, descending=True, stable=True) if k else (d, d)
    top = top[:, :k] - log_z[:, None]
    ids = torch.where(top > -math.inf, ids[:, :k], -1).to(torch.int32)
    return given, entropy, ids, top


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "logprobs":
        R, V, k = case["rows"], case["vocab"], case["top_k"]
        return {"bytes": R * V * size + R * (12 + 8 * k), "flops": 5 * R * V}
    ctx, new = _lengths(case)
    H, heads, d = case["kv_heads"], case["heads"], case["d"]
    pages = int(((ctx + BS - 1) // BS).sum())
    T = int(new.sum())
    if case["op"] == "append":
        touched = int(((ctx - 1) // BS - (ctx - new) // BS + 1).sum())
        return {"bytes": 2 * T * H * d * (size + 1) + touched * (8 * H + 4), "flops": 4 * T * H * d}
    cache = int(ctx.sum()) * H * d * 2 + pages * (8 * H + 4)
    if case["op"] == "decode":
        seen = int(ctx.sum())
    else:
        seen = int((new * (ctx - new) + new * (new + 1) // 2).sum())
    return {"bytes": cache + 2 * T * heads * d * size, "flops": 4 * heads * d * seen}


# ---- the definitions in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_attention(case, s)


def _exact_logprobs(s):
    given, entropy, top = [], [], []
    for x, t in zip(s["logits"].split(64), s["ids"].long().split(64)):
        x = x.double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        p = lp.exp()
        given.append(lp[torch.arange(len(t), device=DEV), t])
        entropy.append(-torch.where(p > 0, p * lp, 0.0).sum(1))
        top.append(torch.topk(lp, s["top_k"], dim=1).values)
    return torch.cat(given), torch.cat(entropy), None, torch.cat(top)


def _e4m3_values():
    """The non-negative e4m3 values in order of their codes 0..126."""
    c = torch.arange(127, device=DEV)
    e, m = c // 8, (c % 8).double()
    return torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.ldexp(torch.ones_like(m), e - 7))


def _exact_round(x, fmt):
    if fmt == "i8":
        lo = torch.floor(x)
        f = x - lo
        up = (f > 0.5) | ((f == 0.5) & (torch.remainder(lo, 2) == 1))
        return lo + up.double()
    grid = _e4m3_values()
    a = x.abs()
    i = torch.searchsorted(grid, a, right=True) - 1
    j = (i + 1).clamp(max=126)
    below, above = a - grid[i], grid[j] - a
    up = (above < below) | ((above == below) & (i % 2 == 1))
    return torch.copysign(torch.where(up, grid[j], grid[i]), x)


def _exact_append(case, s):
    """Block by block of each sequence, from the rows' definition."""
    fmt = case["fmt"]
    ctx, new = _lengths(case)
    cu = np.concatenate([[0], np.cumsum(new)])
    outs = []
    for cache, scale, x in ((s["kc"], s["ks"], s["key"]), (s["vc"], s["vs"], s["value"])):
        val, sc = cache.double(), scale.double()
        for b in range(len(ctx)):
            L, p = int(ctx[b]), int(ctx[b] - new[b])
            ids = s["tables"][b].long()
            while p < L:
                # full blocks together, a block that begins or ends inside a block alone
                whole = p % BS == 0 and L - p >= BS
                n = (L - p) // BS if whole else 1
                o = p % BS
                rows = BS if whole else min(BS - o, L - p)
                at = ids[p // BS:p // BS + n]
                t0 = int(cu[b]) + p - int(ctx[b] - new[b])
                r = x[t0:t0 + n * rows].double().reshape(n, rows, case["kv_heads"], -1).permute(0, 2, 1, 3)
                a = r.abs().amax((2, 3))
                e = torch.floor(torch.log2(a.clamp(min=2.0 ** -130))).long() - 10
                to = torch.ldexp(torch.ones_like(a), e)
                for _ in range(6):
                    to = torch.where(QMAX[fmt] * to < a, 2 * to, to)
                to = to.clamp(min=2.0 ** -126)
                if o:
                    to = torch.maximum(to, sc[at])
                    held = val[at, :, :o] * (sc[at] / to)[..., None, None]
                    val[at, :, :o] = _exact_round(held, fmt)
                val[at, :, o:o + rows] = _exact_round(r / to[..., None, None], fmt)
                sc[at] = to
                p += n * rows
        outs.append((None if fmt == "i8" else val, sc))
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1]


def _exact_attention(case, s):
    ctx, new = _lengths(case)
    cu = np.concatenate([[0], np.cumsum(new)])
    r, out = s["n_rep"], torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(len(ctx)):
        L, n = int(ctx[b]), int(new[b])
        ids = s["tables"][b, :(L + BS - 1) // BS].long()
        for h in range(case["kv_heads"]):
            k = (_raw(s["kc"])[ids, h].view(s["kc"].dtype).double() * s["ks"][ids, h].double()[:, None, None]).reshape(-1, case["d"])[:L]
            v = (_raw(s["vc"])[ids, h].view(s["vc"].dtype).double() * s["vs"][ids, h].double()[:, None, None]).reshape(-1, case["d"])[:L]
            q = s["q"][int(cu[b]):int(cu[b]) + n, h * r:(h + 1) * r].double()
            score = torch.einsum("ird,jd->irj", q, k) * s["scale"]
            ahead = torch.arange(L, device=DEV)[None, :] > (L - n + torch.arange(n, device=DEV))[:, None]
            score = score.masked_fill(ahead[:, None, :], -math.inf)
            w = torch.softmax(score, 2)
            out[int(cu[b]):int(cu[b]) + n, h * r:(h + 1) * r] = torch.einsum("irj,jd->ird", w, v)
    return out
