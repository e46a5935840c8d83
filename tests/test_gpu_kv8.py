"""The 8-bit KV cache on the GPU: append, decode and prefill against plain 64-bit forms.

The append is compared code by code: its scales are powers of two, so every quotient is exact and
there is one right answer. Attention is held to the element-wise bound of _kv8.attention_ref plus
half a step of the output type."""

import math

import numpy as np
import pytest
import torch

from flour_b200 import FlourAttnError, _lib, ops

import _kv8
from _kv8 import FMTS, append_ref, assert_close, attention_ref, inv_sqrt, make_tables, random_pool

pytestmark = pytest.mark.gpu

U16 = 2.0 ** -11  # half a step of f16, relative: how the decode rounds probabilities


def gen_of(device, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def i32(x, device):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=device)


def run_append(pool, key, value, bt, ctx, new, device, one=False, **kw):
    cu = None if one else i32(np.concatenate([[0], np.cumsum(new)]), device)
    ops.paged_append_kv8(*pool, key, value, i32(bt, device), i32(ctx, device), cu, **kw)


def check_append(pool, before, key, value, bt, ctx, new):
    """pool after the call against append_ref on `before` (clones from before the call)."""
    for c, s, c0, s0, x in ((pool[0], pool[2], before[0], before[2], key),
                            (pool[1], pool[3], before[1], before[3], value)):
        raw = c0.view(torch.uint8).cpu().numpy().copy()
        sc = s0.cpu().numpy().copy()
        append_ref(raw, sc, c.dtype, x.double().cpu().numpy(), bt, ctx, new)
        np.testing.assert_array_equal(s.cpu().numpy(), sc)
        got = c.view(torch.uint8).cpu().numpy()
        if c.dtype == torch.float8_e4m3fn:  # NaN's sign is not pinned
            raw, got = [np.where((a & 0x7F) == 0x7F, 0x7F, a) for a in (raw, got)]
        np.testing.assert_array_equal(got, raw)


def clone(pool):
    return [t.clone() for t in pool]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads, d, bs", [(8, 128, 16), (2, 64, 16), (3, 40, 16), (4, 128, 8), (1, 256, 32),
                                          (5, 6, 4)])
def test_append_prompts(device, fmt, dtype, heads, d, bs):
    ctx, new = [1, 15, 16, 17, 33, 200, 64, 5], [1, 15, 16, 1, 18, 200, 16, 0]
    bt, nb = make_tables(ctx, bs, 1)
    g = gen_of(device, 2)
    pool = random_pool(nb, heads, bs, d, fmt, g, device)
    T = sum(new)
    key = (torch.randn((T, heads, d), device=device, generator=g) * 3).to(dtype)
    value = torch.randn((T, heads, d), device=device, generator=g).to(dtype)
    before = clone(pool)
    run_append(pool, key, value, bt, ctx, new, device)
    check_append(pool, before, key, value, bt, ctx, new)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads, d", [(4, 128), (2, 64), (3, 24)])
def test_append_token_by_token_grows_the_scale(device, fmt, heads, d):
    # 40 steps of one token each, louder and quieter in turns, starting on reused blocks.
    S = 3
    bt, nb = make_tables([48] * S, 16, 3)
    g = gen_of(device, 4)
    pool = random_pool(nb, heads, 16, d, fmt, g, device)
    one = True
    for step in range(40):
        ctx = [step + 1, step + 5, step + 8]
        loud = 2.0 ** ((step * 7) % 11 - 5)
        key = (torch.randn((S, heads, d), device=device, generator=g) * loud).to(torch.bfloat16)
        value = torch.zeros_like(key) if step == 16 else key.flip(0).contiguous()
        before = clone(pool)
        run_append(pool, key, value, bt, ctx, [1] * S, device, one=one)
        check_append(pool, before, key, value, bt, ctx, [1] * S)
        one = not one  # the one-token and the varlen form in turns
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_append_values_at_the_borders(device, fmt):
    # Largest codes exactly, halfway cases, the floor of the scale, f32 extremes, zeros.
    d = 128
    top = _kv8.QMAX[fmt]
    rows = [torch.full((d,), top), torch.full((d,), math.nextafter(top, math.inf) * (1 + 1e-6)),
            torch.linspace(-top, top, d), torch.arange(d) + 0.5, torch.zeros(d), torch.full((d,), 1e-45),
            torch.full((d,), 3.4e38), torch.full((d,), -1.2e-38),
            torch.tensor([0.0009765625 * (i + 1) for i in range(d)])]
    x = torch.stack([r.float() for r in rows])[:, None, :].to(device)
    T = len(rows)
    for new, ctx in (([T], [T]), ([1] * T, list(range(1, T + 1)))):
        bt, nb = make_tables(ctx, 16, 5)
        pool = random_pool(nb, 1, 16, d, fmt, gen_of(device, 6), device)
        before = clone(pool)
        run_append(pool, x, -x, bt, ctx, new, device)
        check_append(pool, before, x, -x, bt, ctx, new)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt, ratio", [(torch.int8, 1 / 6), (torch.float8_e4m3fn, 17 / 208)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 40])
def test_append_into_blocks_of_any_scale(device, fmt, ratio, dtype, d):
    # Part-filled blocks of a cache quantised elsewhere, scales that are not powers of two: one
    # sequence whose scale stays, with new values next to the borders between two codes, and one
    # whose scale grows by 1 / ratio, which brings old codes next to such borders.
    H, ctx, new = 3, [14, 14], [7, 7]
    bt, nb = make_tables([16, 16], 16, 62)
    g = gen_of(device, 62)
    top = _kv8.QMAX[fmt]
    pool = random_pool(nb, H, 16, d, fmt, g, device)
    stays, grows = float(np.float32(0.0123)), float(np.float32(ratio)) * 2.0 ** -5
    for s in pool[2:]:
        s[int(bt[0, 0])], s[int(bt[1, 0])] = stays, grows
    key = torch.randn((14, H, d), device=device, generator=g, dtype=torch.float64)
    # The scale stays up to its largest code times 2^-7, the power of two below it: 80 and 284 codes.
    if fmt == torch.int8:
        codes = torch.randint(-80, 80, (7, H, d), device=device, generator=g) + 0.5
    else:  # 5 significant bits, at most 248
        codes = (torch.randint(8, 16, (7, H, d), device=device, generator=g) * 2 + 1) * \
            torch.exp2(torch.randint(-4, 4, (7, H, d), device=device, generator=g).double())
    key[:7] = codes * stays
    key[7:] *= 0.25 * top * 2.0 ** -5 / key[7:].abs().amax((0, 2), keepdim=True)
    key[7:, :, 0] = 0.9 * top * 2.0 ** -5  # the new scale is 2^-5
    key = key.to(dtype)
    before = clone(pool)
    run_append(pool, key, -key, bt, ctx, new, device)
    assert (pool[2][int(bt[0, 0])] == stays).all() and (pool[2][int(bt[1, 0])] == 2.0 ** -5).all()
    check_append(pool, before, key, -key, bt, ctx, new)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_append_nonfinite_values_are_reported_and_do_not_set_the_scale(device, fmt):
    bt, nb = make_tables([20], 16, 7)
    g = gen_of(device, 8)
    pool = random_pool(nb, 2, 16, 64, fmt, g, device)
    key = torch.randn((20, 2, 64), device=device, generator=g).to(torch.bfloat16)
    value = key.clone()
    key[3, 0, 5], key[4, 1, 6], key[17, 0, 0] = math.inf, math.nan, -math.inf
    key[18:, 1] = math.nan
    before = clone(pool)
    ops.device_status()
    run_append(pool, key, value, bt, [20], [20], device)
    assert ops.device_status() == _lib.FA_DEVERR_VALUE
    check_append(pool, before, key, value, bt, [20], [20])


def test_append_strides(device):
    # The (1, Hkv, n, d) layout (token stride d, head stride n d) and a slice of fused qkv rows.
    g = gen_of(device, 9)
    n, H, d = 37, 4, 128
    bt, nb = make_tables([n], 16, 10)
    qkv = torch.randn((n, 8 + 2 * H, d), device=device, generator=g).to(torch.bfloat16)
    key, value = qkv[:, 8:8 + H], torch.randn((H, n, d), device=device, generator=g).to(torch.bfloat16).transpose(0, 1)
    odd = torch.randn((n * H * d + 1,), device=device, generator=g).to(torch.bfloat16)[1:].view(n, H, d)
    for k, v in ((key, value), (odd, key)):  # `odd` starts 2 bytes past an aligned address
        pool = random_pool(nb, H, 16, d, torch.int8, g, device)
        before = clone(pool)
        run_append(pool, k, v, bt, [n], [n], device)
        check_append(pool, before, k, v, bt, [n], [n])


def test_append_leaves_everything_else_alone(device):
    # Bad lengths, bad ids, padded rows behind the last sequence, an empty batch.
    g = gen_of(device, 11)
    ctx, new = [10, 4, 30, 12], [10, 5, 8, 12]   # sequence 1: more new tokens than its length
    bt, nb = make_tables([16, 16, 32, 16], 16, 12)
    bt[2, 1] = nb + 5                             # sequence 2's second block
    pool = random_pool(nb, 2, 16, 64, torch.float8_e4m3fn, g, device)
    key = torch.randn((sum(new) + 9, 2, 64), device=device, generator=g).to(torch.float16)
    key[sum(new):] = math.nan                     # padding
    before = clone(pool)
    ops.device_status()
    run_append(pool, key, key, bt, ctx, new, device)
    assert ops.device_status() == _lib.FA_DEVERR_CONTEXT | _lib.FA_DEVERR_BLOCK_ID
    for c, s, c0, s0 in ((pool[0], pool[2], before[0], before[2]), (pool[1], pool[3], before[1], before[3])):
        raw, sc = c0.view(torch.uint8).cpu().numpy().copy(), s0.cpu().numpy().copy()
        x = key.double().cpu().numpy()
        append_ref(raw, sc, c.dtype, x[:10], bt[:1], [10], [10])
        append_ref(raw, sc, c.dtype, x[23:35], bt[3:], [12], [12])
        np.testing.assert_array_equal(s.cpu().numpy(), sc)
        np.testing.assert_array_equal(c.view(torch.uint8).cpu().numpy(), raw)
    run_append(pool, key[:0], key[:0], bt, ctx, [0, 0, 0, 0], device)
    assert ops.device_status() == 0
    # A cu_seqlens entry past the packed tokens is reported, and nothing of that sequence written.
    after = clone(pool)
    ops.paged_append_kv8(*pool, key[:8], key[:8], i32(bt[:2], device), i32([10, 20], device),
                         i32([0, 4, 11], device))
    assert ops.device_status() == _lib.FA_DEVERR_SEQLEN
    assert torch.equal(pool[2][int(bt[1, 0])], after[2][int(bt[1, 0])])


def decode_case(device, fmt, dtype, Hq, Hkv, d, ctx, seed, bs=16, q_scale=1.0, kernel_u=U16):
    bt, nb = make_tables(ctx, bs, seed)
    g = gen_of(device, seed)
    pool = random_pool(nb, Hkv, bs, d, fmt, g, device)
    q = (torch.randn((len(ctx), Hq, d), device=device, generator=g) * q_scale).to(dtype)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [1] * len(ctx),
                              Hq // Hkv, inv_sqrt(d), kernel_u)
    return pool, q, i32(bt, device), i32(ctx, device), want, tol


def run_decode(pool, q, bt, cl, ctx, Hkv, ws=None, **kw):
    return ops.paged_decode_kv8(q, *pool, bt, cl, q.shape[1] // Hkv, inv_sqrt(q.shape[2]), int(max(ctx)),
                                ws or ops.Workspace(), **kw)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq, Hkv, d", [(32, 8, 128), (28, 4, 128), (14, 2, 64), (8, 8, 128), (8, 1, 64)])
@pytest.mark.parametrize("ctx", [[1], [15, 16, 17, 31, 32, 33], [511, 2, 1200, 513]])
def test_decode(device, fmt, dtype, Hq, Hkv, d, ctx):
    pool, q, bt, cl, want, tol = decode_case(device, fmt, dtype, Hq, Hkv, d, ctx, 20)
    assert_close(run_decode(pool, q, bt, cl, ctx, Hkv), want, tol)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype, Hq, Hkv, d, bs", [
    (torch.float32, 8, 2, 128, 16), (torch.float32, 14, 2, 64, 16), (torch.bfloat16, 16, 1, 128, 16),
    (torch.float16, 6, 3, 96, 8), (torch.float32, 4, 4, 6, 4), (torch.bfloat16, 4, 2, 256, 32)])
def test_decode_other_shapes(device, fmt, dtype, Hq, Hkv, d, bs):
    ctx = [1, bs, bs + 1, 300]
    pool, q, bt, cl, want, tol = decode_case(device, fmt, dtype, Hq, Hkv, d, ctx, 21, bs=bs, kernel_u=0.0)
    assert_close(run_decode(pool, q, bt, cl, ctx, Hkv), want, tol)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_decode_long_context_splits(device, fmt):
    ctx = [9001, 4097, 12345]
    pool, q, bt, cl, want, tol = decode_case(device, fmt, torch.bfloat16, 8, 2, 128, ctx, 22)
    ws = ops.Workspace()
    out = run_decode(pool, q, bt, cl, ctx, 2, ws)
    assert_close(out, want, tol)
    assert torch.equal(out, run_decode(pool, q, bt, cl, ctx, 2, ws))


def test_decode_scales_that_differ_from_page_to_page(device):
    # Scales over 2^+-24 that are not powers of two: accumulators of neighbouring pages differ.
    ctx = [400, 37]
    pool, q, bt, cl, _, _ = decode_case(device, torch.int8, torch.bfloat16, 8, 2, 128, ctx, 23)
    g = gen_of(device, 24)
    pool = (pool[0], pool[1], pool[2] * 1.37, torch.exp2(torch.rand_like(pool[3]) * 48 - 24))
    want, tol = attention_ref(q.double().cpu().numpy(), pool, bt, ctx, [1, 1], 4, inv_sqrt(128), U16)
    assert_close(run_decode(pool, q, bt, cl, ctx, 2), want, tol)


@pytest.mark.parametrize("first, second", [(2.0 ** -12, 2.0 ** -6), (2.0 ** -6, 2.0 ** -12), (0.02, 0.0007),
                                           (1e-33, 1e-34), (3e-35, 2e-35)])
def test_decode_small_probabilities_of_a_quiet_page(device, first, second):
    # Two pages of one step, the scales of V up to 64 apart, and probabilities of all sizes: those
    # of the quiet page must keep their bits.
    ctx = [17 + s % 16 for s in range(60)]
    pool, q, bt, cl, _, _ = decode_case(device, torch.float8_e4m3fn, torch.float16, 8, 2, 128, ctx, 46,
                                        q_scale=3.0)
    pool[3][bt[:, 0].long()] = first
    pool[3][bt[:, 1].long()] = second
    want, tol = attention_ref(q.double().cpu().numpy(), pool, bt, ctx, [1] * 60, 4, inv_sqrt(128), U16)
    out = run_decode(pool, q, bt, cl, ctx, 2)
    assert_close(out, want, tol)
    out = run_decode(pool, q.to(torch.bfloat16), bt, cl, ctx, 2)
    want, tol = attention_ref(q.to(torch.bfloat16).double().cpu().numpy(), pool, bt, ctx, [1] * 60, 4,
                              inv_sqrt(128), U16)
    assert_close(out, want, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("first, second", [(2.0 ** 6, 2.0 ** -14), (2.0 ** -14, 2.0 ** 6), (0.9, 0.0007),
                                           (0.0007, 0.9), (2.0 ** -126, 2.0 ** -112), (1.3e-34, 1.7e-36)])
def test_decode_small_probabilities_of_a_loud_page(device, dtype, first, second):
    # Two pages of one step, the scales of V more than 64 apart, and the louder page's probabilities
    # near 2^-22 of the largest: its scale multiplies their rounding. Probabilities are rounded at
    # 2^12 times their size, so under the smallest normal f16 they move in half steps of 2^-37.
    ctx, d, Hkv, n_rep = [32, 29, 32], 128, 2, 4
    bt, nb = make_tables(ctx, 16, 60)
    g = gen_of(device, 60)
    pool = random_pool(nb, Hkv, 16, d, torch.int8, g, device)
    loud = 0 if first > second else 1
    k = torch.randint(-8, 9, pool[0].shape, device=device, generator=g, dtype=torch.int8)
    k[..., 0] = 127
    k[torch.as_tensor(bt[:, loud], device=device).long(), :, :, 0] = 0
    scales = torch.empty_like(pool[3])
    scales[torch.as_tensor(bt[:, 0], device=device).long()] = first
    scales[torch.as_tensor(bt[:, 1], device=device).long()] = second
    pool = (k, pool[1], torch.full_like(pool[2], 1 / 64.0), scales)
    q = torch.randn((3, Hkv * n_rep, d), device=device, generator=g)
    q[..., 0] = 22 * math.log(2.0) / (127 / 64.0 * inv_sqrt(d))
    q = q.to(dtype)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [1] * 3, n_rep,
                              inv_sqrt(d), U16)
    v = np.abs(_kv8.dequant(pool[1], pool[3]))
    for s, L in enumerate(ctx):  # sum |v| over a sequence's tokens, a row for each query head
        total = np.concatenate([v[b] for b in bt[s]], 1)[:, :L].sum(1).repeat(n_rep, 0)
        tol[s] += (2.0 ** -37 - 2.0 ** -24) * total
    out = run_decode(pool, q, i32(bt, device), i32(ctx, device), ctx, Hkv)
    assert_close(out, want, tol)
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_scale", [2.0 ** -60, 2.0 ** 40, 0.0])
def test_decode_queries_outside_f16(device, q_scale):
    ctx = [100]
    bt, nb = make_tables(ctx, 16, 25)
    pool = random_pool(nb, 2, 16, 64, torch.float8_e4m3fn, gen_of(device, 25), device)
    pool = (pool[0], pool[1], pool[2] / (q_scale or 1.0), pool[3])
    q = (torch.randn((1, 4, 64), device=device, generator=gen_of(device, 26)) * q_scale).to(torch.bfloat16)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [1], 2, inv_sqrt(64), U16)
    assert_close(run_decode(pool, q, i32(bt, device), i32(ctx, device), ctx, 2), want, tol)


def poison_tails(pool, bt, ctx):
    """NaN codes behind each sequence's last token, NaN scales in blocks nobody holds."""
    bs = pool[0].shape[2]
    used = set()
    for s, L in enumerate(ctx):
        n = (L + bs - 1) // bs
        used |= {int(b) for b in bt[s, :n]}
        if L % bs:
            for c in pool[:2]:
                c.view(torch.uint8)[int(bt[s, n - 1]), :, L % bs:] = 0x7F
    for b in set(range(pool[0].shape[0])) - used:
        pool[2][b] = math.nan
        pool[3][b] = math.nan


@pytest.mark.parametrize("Hq, Hkv, d, dtype", [(32, 8, 128, torch.bfloat16), (14, 2, 64, torch.float16),
                                               (4, 2, 96, torch.float32)])
def test_stale_nan_behind_the_context_is_not_seen(device, Hq, Hkv, d, dtype):
    ctx, new = [1, 17, 47, 130, 16], [1, 2, 30, 130, 5]
    bt, nb = make_tables(ctx, 16, 27)
    g = gen_of(device, 27)
    pool = random_pool(nb, Hkv, 16, d, torch.float8_e4m3fn, g, device)
    poison_tails(pool, bt, ctx)
    q = torch.randn((sum(new), Hq, d), device=device, generator=g).to(dtype)
    first = np.cumsum([0] + new[:-1])
    want, tol = attention_ref(q.double().cpu().numpy()[first], pool, torch.as_tensor(bt), ctx, [1] * 5,
                              Hq // Hkv, inv_sqrt(d), U16)
    assert_close(run_decode(pool, q[first].contiguous(), i32(bt, device), i32(ctx, device), ctx, Hkv), want, tol)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, Hq // Hkv,
                              inv_sqrt(d), 2.0 ** -8)
    assert_close(run_prefill(pool, q, bt, ctx, new, Hkv, device), want, tol)
    assert ops.device_status() == 0


def run_prefill(pool, q, bt, ctx, new, Hkv, device, ws=None, slack=0, **kw):
    bs = pool[0].shape[2]
    cu = i32(np.concatenate([[0], np.cumsum(new)]), device)
    blocks = sum((c + bs - 1) // bs for c in ctx) + slack
    return ops.paged_prefill_kv8(q, *pool, cu, i32(ctx, device), i32(bt, device), q.shape[1] // Hkv,
                                 inv_sqrt(q.shape[2]), int(max(new)), int(max(ctx)), blocks,
                                 ws or ops.Workspace(), **kw)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq, Hkv, d", [(8, 2, 128), (7, 1, 128), (14, 2, 64)])
@pytest.mark.parametrize("ctx, new", [
    ([300, 90, 257], [236, 90, 129]),       # cached prefixes, ragged ends
    ([1], [1]),                             # one token (the decode)
    ([40, 700], [0, 3]),                    # fewer rows than one query tile; an empty sequence
    ([64, 1, 33, 500], [1, 1, 1, 1]),       # one each
    ([129], [128]),
])
def test_prefill(device, fmt, dtype, Hq, Hkv, d, ctx, new):
    bt, nb = make_tables(ctx, 16, 30)
    g = gen_of(device, 30)
    pool = random_pool(nb, Hkv, 16, d, fmt, g, device)
    q = torch.randn((sum(new), Hq, d), device=device, generator=g).to(dtype)
    # bf16 prompts round probabilities to bf16 (half a step: 2^-8)
    u = 0.0 if dtype == torch.float32 else (2.0 ** -8 if dtype == torch.bfloat16 else U16)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, Hq // Hkv,
                              inv_sqrt(d), u)
    assert_close(run_prefill(pool, q, bt, ctx, new, Hkv, device, slack=5), want, tol)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq, Hkv, ctx, new", [
    (8, 2, [3000], [40]),                    # one chunk over many parts
    (7, 1, [1500], [1400]),                  # chunks that end in early parts
    (8, 1, [2500, 129, 700, 1], [3, 129, 70, 1]),  # short sequences beside a long one
    (16, 1, [5000], [9]),                    # n_rep 16: fewer rows than one query tile
])
def test_prefill_split_over_the_context(device, dtype, Hq, Hkv, ctx, new):
    bt, nb = make_tables(ctx, 16, 44)
    g = gen_of(device, 44)
    pool = random_pool(nb, Hkv, 16, 128, torch.float8_e4m3fn, g, device)
    poison_tails(pool, bt, ctx)
    q = torch.randn((sum(new) + 5, Hq, 128), device=device, generator=g).to(dtype)
    out = torch.full_like(q, 7.0)
    ws = ops.Workspace()
    for _ in range(2):
        run_prefill(pool, q, bt, ctx, new, Hkv, device, ws=ws, out=out)
        want, tol = attention_ref(q[:sum(new)].double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new,
                                  Hq // Hkv, inv_sqrt(128), 2.0 ** -8 if dtype == torch.bfloat16 else U16)
        assert_close(out[:sum(new)], want, tol)
        assert (out[sum(new):] == 7.0).all()
    assert ops.device_status() == 0
    # A refused sequence (its blocks do not fit) is zeroed, the others stand.
    if len(ctx) > 1:
        run_prefill(pool, q, bt, ctx, new, Hkv, device, ws=ws, out=out, slack=-1)
        assert ops.device_status() == _lib.FA_DEVERR_CONTEXT
        assert not out[sum(new) - 1].any()
        assert_close(out[:sum(new) - 1], want[:-1], tol[:-1])


def test_prefill_equals_the_16_bit_prefill_of_the_same_values(device):
    # Power-of-two scales make the bf16 copy exact, so both prefills see one cache.
    ctx, new = [400, 129, 1000], [400, 60, 513]
    bt, nb = make_tables(ctx, 16, 31)
    g = gen_of(device, 31)
    for fmt in FMTS:
        pool = random_pool(nb, 8, 16, 128, fmt, g, device)
        q = torch.randn((sum(new), 32, 128), device=device, generator=g).to(torch.bfloat16)
        out = run_prefill(pool, q, bt, ctx, new, 8, device)
        kc, vc = [(c.float() * s[:, :, None, None]).to(torch.bfloat16) for c, s in zip(pool[:2], pool[2:])]
        cu = i32(np.concatenate([[0], np.cumsum(new)]), device)
        want = ops.paged_prefill(q, kc, vc, cu, i32(ctx, device), i32(bt, device), 4, inv_sqrt(128),
                                 max(new), max(ctx), ops.Workspace())
        assert torch.equal(out, want)


def test_prefill_refuses_sequences_past_total_blocks(device):
    ctx = [64, 200, 32]
    bt, nb = make_tables(ctx, 16, 32)
    g = gen_of(device, 32)
    pool = random_pool(nb, 2, 16, 128, torch.int8, g, device)
    q = torch.randn((sum(ctx), 8, 128), device=device, generator=g).to(torch.bfloat16)
    want = run_prefill(pool, q, bt, ctx, ctx, 2, device)
    ops.device_status()
    out = run_prefill(pool, q, bt, ctx, ctx, 2, device, slack=-3)
    assert ops.device_status() == _lib.FA_DEVERR_CONTEXT
    # 4 + 13 + 2 pages against 16 blocks: the first sequence fits, packing ends at the second.
    assert torch.equal(out[:64], want[:64])
    assert not out[64:].any()


def test_prefill_rows_behind_the_last_sequence_stay(device):
    ctx = [100, 60]
    bt, nb = make_tables(ctx, 16, 33)
    g = gen_of(device, 33)
    pool = random_pool(nb, 2, 16, 128, torch.float8_e4m3fn, g, device)
    q = torch.randn((200, 8, 128), device=device, generator=g).to(torch.bfloat16)
    q[160:] = math.nan
    out = torch.full_like(q, 7.0)
    run_prefill(pool, q, bt, ctx, ctx, 2, device, out=out)
    assert (out[160:] == 7.0).all()
    want, tol = attention_ref(q[:160].double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, ctx, 4,
                              inv_sqrt(128), 2.0 ** -8)
    assert_close(out[:160], want, tol)


@pytest.mark.parametrize("Hq, Hkv, d, dtype, S, hi", [
    (8, 2, 128, torch.bfloat16, 9, 300), (14, 2, 64, torch.float16, 900, 40), (4, 2, 40, torch.float32, 9, 60)])
def test_prefill_of_at_most_one_token_each(device, Hq, Hkv, d, dtype, S, hi):
    # Every third sequence has no new token (some of those no context either), so a row's number is
    # not its sequence's; the batch is padded to one row per sequence.
    rng = np.random.default_rng(35)
    ctx = rng.integers(1, hi, S).tolist()
    new = [0 if s % 3 == 0 else 1 for s in range(S)]
    ctx[3] = 0
    bt, nb = make_tables(ctx, 16, 35)
    g = gen_of(device, 35)
    pool = random_pool(nb, Hkv, 16, d, torch.float8_e4m3fn, g, device)
    q = torch.randn((S, Hq, d), device=device, generator=g).to(dtype)
    rows = sum(new)
    q[rows:] = math.nan
    out = torch.full_like(q, 7.0)
    ops.device_status()
    cu = i32(np.concatenate([[0], np.cumsum(new)]), device)
    ops.paged_prefill_kv8(q, *pool, cu, i32(ctx, device), i32(bt, device), Hq // Hkv, inv_sqrt(d), 1, max(ctx),
                          nb, ops.Workspace(), out)
    assert ops.device_status() == 0
    ctx[3] = 1  # no row of it is compared
    want, tol = attention_ref(q[:rows].double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, Hq // Hkv,
                              inv_sqrt(d), 0.0 if dtype == torch.float32 else U16)
    assert_close(out[:rows], want, tol)
    assert (out[rows:] == 7.0).all()


def test_prefill_of_one_token_each_reports_more(device):
    ctx = [40, 50, 60]
    bt, nb = make_tables(ctx, 16, 36)
    g = gen_of(device, 36)
    pool = random_pool(nb, 2, 16, 128, torch.int8, g, device)
    q = torch.randn((3, 8, 128), device=device, generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    ops.device_status()
    ops.paged_prefill_kv8(q, *pool, i32([0, 2, 2, 3], device), i32(ctx, device), i32(bt, device), 4, inv_sqrt(128),
                          1, 60, nb, ops.Workspace(), out)
    assert ops.device_status() == _lib.FA_DEVERR_SEQLEN
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [2, 0, 1], 4,
                              inv_sqrt(128), U16)
    assert_close(out[2:], want[2:], tol[2:])
    assert (out[:2] == 7.0).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_prefill_of_the_largest_f16_values(device, fmt):
    # 65504 rounds to 65536 in both formats, which f16 does not hold. Equal keys: means of values.
    ctx, new = [70], [70]
    bt, nb = make_tables(ctx, 16, 37)
    g = gen_of(device, 37)
    pool = random_pool(nb, 2, 16, 128, fmt, g, device)
    key = torch.full((70, 2, 128), 65504.0, dtype=torch.float16, device=device)
    value = torch.randn((70, 2, 128), device=device, generator=g).half()
    value[:, 1] = -65504.0
    run_append(pool, key, value, bt, ctx, new, device)
    q = (torch.randn((70, 8, 128), device=device, generator=g) * 2.0 ** -10).half()
    out = run_prefill(pool, q, bt, ctx, new, 2, device)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, 4, inv_sqrt(128),
                              2.0 ** -8)
    assert_close(out[:, :4], want[:, :4], tol[:, :4])
    np.testing.assert_allclose(want[:, 4:], -65536.0, rtol=1e-12)  # 70 sums in 64 bits
    # The copy's -65504 times probabilities rounded to f16, both ways and twice (P, then 1 / l).
    err = (out[:, 4:].double() + 65504.0).abs()
    assert err.max() <= 65504.0 * 2.0 ** -9
    # The decode's and the generic kernel's f32 sums are -65536: the largest f16, not an infinity.
    one = run_decode(pool, q[:1], i32(bt, device), i32(ctx, device), ctx, 2)
    assert (one[:, 4:] == -65504.0).all()
    slow = ops.paged_prefill_kv8(q, *pool, i32([0, 70], device), i32(ctx, device), i32(bt, device), 4,
                                 inv_sqrt(128), 70, 70, 0, ops.Workspace())
    assert (slow[:, 4:] == -65504.0).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("ctx, new", [([128], [128]), ([2944], [40])])  # in one piece, split over the context
def test_prefill_f16_outputs_saturate(device, ctx, new):
    # Values of 65504, one key of each 128 with probability 1 and the others just above the middle
    # of two f16 numbers at 0.5: rounded up, they carry the mean to 65534, which f16 rounds to inf.
    H, n_rep, d = 2, 4, 128
    bt, nb = make_tables(ctx, 16, 61)
    g = gen_of(device, 61)
    pool = random_pool(nb, H, 16, d, torch.float8_e4m3fn, g, device)
    key = torch.zeros((ctx[0], H, d), dtype=torch.float16, device=device)
    key[::128, :, 0] = 1.0
    value = torch.full_like(key, 65504.0)
    value[:, 1] = -65504.0
    run_append(pool, key, value, bt, ctx, ctx, device)
    q = torch.zeros((new[0], H * n_rep, d), dtype=torch.float16, device=device)
    q[..., 0] = 1.0
    scale = math.log(2.0) - 1.05 * 2.0 ** -11  # e^-scale = 0.5 (1 + 1.05 * 2^-11)
    out = ops.paged_prefill_kv8(q, *pool, i32([0, new[0]], device), i32(ctx, device), i32(bt, device), n_rep,
                                scale, new[0], ctx[0], nb, ops.Workspace())
    assert (out[:, :n_rep] == 65504.0).all() and (out[:, n_rep:] == -65504.0).all()
    assert ops.device_status() == 0


def test_bad_lengths_and_ids_are_reported(device):
    ctx = [40, 50]
    pool, q, bt, cl, want, tol = decode_case(device, torch.int8, torch.bfloat16, 8, 2, 128, ctx, 34)
    ops.device_status()
    out = run_decode(pool, q, bt, i32([0, 50], device), ctx, 2)
    assert ops.device_status() == _lib.FA_DEVERR_CONTEXT
    assert not out[0].any()
    assert_close(out[1:], want[1:], tol[1:])
    bad = bt.clone()
    bad[0, 1] = -3
    run_decode(pool, q, bad, cl, ctx, 2)
    assert ops.device_status() == _lib.FA_DEVERR_BLOCK_ID
    q2 = q.repeat_interleave(20, 0)
    run_prefill(pool, q2, bad.cpu().numpy(), ctx, [20, 20], 2, device)
    assert ops.device_status() == _lib.FA_DEVERR_BLOCK_ID


def test_one_workspace_two_graphs_and_other_calls(device):
    # A decode and a prefill captured on one workspace, replayed between eager calls of other sizes.
    ctx, new = [3000, 2500], [200, 100]
    pool, q, bt, cl, want, tol = decode_case(device, torch.float8_e4m3fn, torch.bfloat16, 8, 2, 128, ctx, 35)
    big_ctx = [600] * 40
    bpool, bq, bbt, bcl, bwant, btol = decode_case(device, torch.int8, torch.bfloat16, 32, 8, 128, big_ctx, 36)
    qp = torch.randn((sum(new), 8, 128), device=device, generator=gen_of(device, 37)).to(torch.bfloat16)
    ws = ops.Workspace()
    ws.get(64 << 20)
    want_p = run_prefill(pool, qp, bt.cpu().numpy(), ctx, new, 2, device)
    cu, blocks = i32([0, 200, 300], device), sum((c + 15) // 16 for c in ctx)
    out_d, out_p = torch.empty_like(q), torch.empty_like(qp)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0], stream=s):
        run_decode(pool, q, bt, cl, ctx, 2, ws, out=out_d)
    with torch.cuda.graph(graphs[1], stream=s):
        ops.paged_prefill_kv8(qp, *pool, cu, cl, bt, 4, inv_sqrt(128), 200, 3000, blocks, ws, out=out_p)
    for _ in range(2):
        for order in ((0, 1), (1, 0)):
            for i in order:
                out_d.zero_()
                out_p.zero_()
                graphs[i].replay()
                if i == 0:
                    assert_close(out_d, want, tol)
                else:
                    assert torch.equal(out_p, want_p)
            assert_close(run_decode(bpool, bq, bbt, bcl, big_ctx, 8, ws), bwant, btol)
    del graphs
    assert ops.device_status() == 0


def test_graphs_of_any_sizes_share_a_workspace(device):
    # Captured largest first: many tickets, then few, then a prefill's copy; replayed in all orders.
    from itertools import permutations
    ws = ops.Workspace()
    ws.get(96 << 20)
    cases, graphs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for Hq, Hkv, ctx, seed in ((32, 8, [700] * 100, 50), (8, 2, [5000, 3000], 51)):
        pool, q, bt, cl, want, tol = decode_case(device, torch.int8, torch.bfloat16, Hq, Hkv, 128, ctx, seed)
        ref = run_decode(pool, q, bt, cl, ctx, Hkv)
        assert_close(ref, want, tol)
        out, g = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run_decode(pool, q, bt, cl, ctx, Hkv, ws, out=out)
        cases.append((out, ref, pool, q, bt, cl))
        graphs.append(g)
    _, _, pool, _, bt, cl = cases[1]
    qp = torch.randn((90, 8, 128), device=device, generator=gen_of(device, 52)).to(torch.bfloat16)
    args = (qp, *pool, i32([0, 50, 90], device), cl, bt, 4, inv_sqrt(128), 50, 5000, 501)
    ref = ops.paged_prefill_kv8(*args, ops.Workspace())
    out, g = torch.empty_like(qp), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ops.paged_prefill_kv8(*args, ws, out=out)
    cases.append((out, ref))
    graphs.append(g)
    for order in permutations(range(3)):
        for i in order:
            cases[i][0].zero_()
            graphs[i].replay()
            assert torch.equal(cases[i][0], cases[i][1]), (order, i)
    del graphs, g
    assert ops.device_status() == 0


def test_a_workspace_grows_under_a_captured_graph(device):
    # A decode captured on a warmed workspace, a prefill that outgrows it, other tensors where its
    # buffer would have been: the replay gives the same bits and touches none of them.
    ctx, new = [3000, 2500], [200, 100]
    pool, q, bt, cl, want, tol = decode_case(device, torch.float8_e4m3fn, torch.bfloat16, 8, 2, 128, ctx, 63)
    qp = torch.randn((300, 8, 128), device=device, generator=gen_of(device, 64)).to(torch.bfloat16)
    ws = ops.Workspace()
    ref = run_decode(pool, q, bt, cl, ctx, 2, ws)
    assert_close(ref, want, tol)
    size, out = ws.get(1).numel(), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_decode(pool, q, bt, cl, ctx, 2, ws, out=out)
    want_p = run_prefill(pool, qp, bt.cpu().numpy(), ctx, new, 2, device)
    assert torch.equal(run_prefill(pool, qp, bt.cpu().numpy(), ctx, new, 2, device, ws=ws), want_p)
    assert ws.get(1).numel() > size
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device=device) for _ in range(8)]
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, ref)
        assert torch.equal(run_prefill(pool, qp, bt.cpu().numpy(), ctx, new, 2, device, ws=ws), want_p)
    assert all((t == 0x5A).all() for t in others)
    del graph
    assert ops.device_status() == 0


def test_graphs_captured_on_a_fresh_workspace(device):
    # No call before the captures, the largest first: graphs are replayed in any order, and eager
    # calls come before the first replay.
    ws, cases = ops.Workspace(), []
    for Hq, Hkv, ctx, seed in ((32, 8, [700] * 100, 65), (8, 2, [5000, 3000], 66), (8, 2, [900], 67)):
        pool, q, bt, cl, want, tol = decode_case(device, torch.int8, torch.bfloat16, Hq, Hkv, 128, ctx, seed)
        ref = run_decode(pool, q, bt, cl, ctx, Hkv)
        assert_close(ref, want, tol)
        out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(2):
                run_decode(pool, q, bt, cl, ctx, Hkv, ws, out=out)
        cases.append((graph, out, ref, (pool, q, bt, cl, ctx, Hkv)))
    for order in ((2, 1), (1, 2, 0), (0, 2, 1)):
        for i in order:
            graph, out, ref, args = cases[i]
            assert torch.equal(run_decode(*args, ws), ref)
            out.zero_()
            graph.replay()
            assert torch.equal(out, ref)
    del graph, cases
    assert ops.device_status() == 0


def test_a_16_bit_workspace_is_refused(device):
    pool, q, bt, cl, _, _ = decode_case(device, torch.int8, torch.bfloat16, 8, 2, 128, [40, 5000], 53)
    ws = ops.Workspace()
    kc = torch.zeros(pool[0].shape, dtype=torch.bfloat16, device=device)
    ops.paged_decode(q, kc, kc, bt, cl, 4, 0.1, 5000, ws)
    with pytest.raises(FlourAttnError):
        ops.paged_decode_kv8(q, *pool, bt, cl, 4, 0.1, 5000, ws)


def test_side_stream_and_append_then_decode_chain(device):
    # One step as a server runs it: prompts appended and attended, then 20 tokens one by one,
    # all on a side stream, against the plain forms on the same codes.
    H, Hq, d = 2, 8, 128
    lens = [37, 5, 64]
    bt, nb = make_tables([c + 20 for c in lens], 16, 40)
    for fmt in FMTS:
        g = gen_of(device, 41)
        pool = random_pool(nb, H, 16, d, fmt, g, device)
        ws = ops.Workspace()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            k, v = (torch.randn((sum(lens), H, d), device=device, generator=g).to(torch.bfloat16) for _ in "kv")
            q = torch.randn((sum(lens), Hq, d), device=device, generator=g).to(torch.bfloat16)
            run_append(pool, k, v, bt, lens, lens, device)
            out = run_prefill(pool, q, bt, lens, lens, H, device, ws=ws)
        side.synchronize()
        want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), lens, lens, 4,
                                  inv_sqrt(d), 2.0 ** -8)
        assert_close(out, want, tol)
        ctx = list(lens)
        for _ in range(20):
            ctx = [c + 1 for c in ctx]
            with torch.cuda.stream(side):
                k, v = (torch.randn((3, H, d), device=device, generator=g).to(torch.bfloat16) for _ in "kv")
                q = torch.randn((3, Hq, d), device=device, generator=g).to(torch.bfloat16)
                run_append(pool, k, v, bt, ctx, [1] * 3, device, one=True)
                out = run_decode(pool, q, i32(bt, device), i32(ctx, device), ctx, H, ws)
            side.synchronize()
            want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [1] * 3, 4,
                                      inv_sqrt(d), U16)
            assert_close(out, want, tol)
        assert ops.device_status() == 0


def test_an_explicit_stream_is_in_order_with_itself(device):
    # stream= another stream than the current one, which stands still meanwhile: workspaces fresh,
    # outgrown and made on the current stream, strided queries, outputs in memory that was in use.
    ctx, new = [3000, 2500], [200, 100]
    pool, q, bt, cl, want, tol = decode_case(device, torch.float8_e4m3fn, torch.bfloat16, 8, 2, 128, ctx, 68)
    cu, blocks = i32([0, 200, 300], device), sum((c + 15) // 16 for c in ctx)
    qp = torch.randn((300, 8, 128), device=device, generator=gen_of(device, 69)).to(torch.bfloat16)
    want_p = run_prefill(pool, qp, bt.cpu().numpy(), ctx, new, 2, device)
    ref = run_decode(pool, q, bt, cl, ctx, 2)
    assert_close(ref, want, tol)
    strided = torch.zeros((2, 8, 256), dtype=torch.bfloat16, device=device)
    strided[..., :128] = q
    logits = torch.randn((3, 5000), device=device)
    ids = i32([1, 2, 3], device)
    ref_l = ops.token_logprobs(logits, ids, 5)
    key = torch.randn((2, 2, 128), device=device).to(torch.bfloat16)
    after = clone(pool)
    ops.paged_append_kv8(*after, key, key, bt, cl)
    side = torch.cuda.Stream()
    for junk_on in (torch.cuda.current_stream(), side):  # what fresh memory holds
        with torch.cuda.stream(junk_on):
            junk = [torch.full((32 << 20,), 0x5A, dtype=torch.uint8, device=device) for _ in range(6)]
            del junk
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(1_000_000_000)  # 0.5 s
    early = ops.Workspace()
    early.get(64 << 20)  # filled behind the sleep
    done.record()
    ws = ops.Workspace()
    got = [run_decode(pool, strided[..., :128], bt, cl, ctx, 2, ws, stream=side) for _ in range(2)]
    got_p = [ops.paged_prefill_kv8(qp, *pool, cu, cl, bt, 4, inv_sqrt(128), 200, 3000, blocks, ws, stream=side)
             for _ in range(2)]
    got.append(run_decode(pool, strided[..., :128], bt, cl, ctx, 2, ws, stream=side))
    got_l = ops.token_logprobs(logits, ids, 5, stream=side)
    ops.paged_append_kv8(*pool, key, key, bt, cl, stream=side)
    side.synchronize()
    assert not done.query()  # none of it waited for the current stream
    with torch.cuda.stream(side):
        assert all(torch.equal(o, ref) for o in got) and all(torch.equal(o, want_p) for o in got_p)
        assert all(torch.equal(a, b) for a, b in zip(got_l, ref_l))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, after))
    late = run_decode(pool, q, bt, cl, ctx, 2, early, stream=side)
    side.synchronize()
    assert done.query()  # the fill it needs is behind the sleep
    assert torch.equal(late, run_decode(pool, q, bt, cl, ctx, 2))
    assert ops.device_status() == 0


@pytest.mark.parametrize("S, ctx_hi", [(500, 40), (1100, 20)])
def test_many_sequences(device, S, ctx_hi):
    # More sequences than one decode launch takes, more than the append searches in shared memory.
    rng = np.random.default_rng(45)
    ctx = rng.integers(1, ctx_hi + 1, S)
    new = np.minimum(rng.integers(0, 4, S), ctx)
    ctx[::7], new[::7] = 2, 2
    bt, nb = make_tables(ctx, 16, 45)
    g = gen_of(device, 45)
    pool = random_pool(nb, 2, 16, 64, torch.int8, g, device)
    T = int(new.sum())
    key, value = (torch.randn((T, 2, 64), device=device, generator=g).to(torch.float16) for _ in "kv")
    before = clone(pool)
    run_append(pool, key, value, bt, ctx, new, device)
    check_append(pool, before, key, value, bt, ctx, new)
    q = torch.randn((S, 8, 64), device=device, generator=g).to(torch.bfloat16)
    want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, [1] * S, 4,
                              inv_sqrt(64), U16)
    assert_close(run_decode(pool, q, i32(bt, device), i32(ctx, device), ctx, 2), want, tol)
    assert ops.device_status() == 0


def test_prefill_of_many_sequences(device):
    # 2049 sequences are more than the copy to 16 bits takes in one call: the generic kernel.
    for S in (300, 2049):
        rng = np.random.default_rng(46)
        ctx = rng.integers(1, 20, S)
        new = np.minimum(rng.integers(0, 3, S), ctx)
        bt, nb = make_tables(ctx, 16, 46)
        g = gen_of(device, 46)
        pool = random_pool(nb, 1, 16, 128, torch.float8_e4m3fn, g, device)
        q = torch.randn((int(new.sum()), 4, 128), device=device, generator=g).to(torch.float16)
        want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, 4,
                                  inv_sqrt(128), U16)
        assert_close(run_prefill(pool, q, bt, ctx, new, 1, device), want, tol)
        assert ops.device_status() == 0


@pytest.mark.parametrize("ctx", [[20000, 5, 17, 90, 1], [31, 4000, 30, 33, 3000], [512] * 9, [513] * 60])
def test_decode_skewed_batches_repeat(device, ctx):
    # One sequence holds nearly all pages, or items end inside and at the ends of the warps' ranges.
    for fmt in FMTS:
        pool, q, bt, cl, want, tol = decode_case(device, fmt, torch.float16, 8, 2, 128, ctx, 47)
        ws = ops.Workspace()
        out = run_decode(pool, q, bt, cl, ctx, 2, ws)
        assert_close(out, want, tol)
        for _ in range(3):  # the same bits whichever CTA joins, and tickets back at zero
            assert torch.equal(run_decode(pool, q, bt, cl, ctx, 2, ws), out)
        # A larger bound than the longest context: the same ranges.
        again = ops.paged_decode_kv8(q, *pool, bt, cl, 4, inv_sqrt(128), bt.shape[1] * 16, ws)
        assert_close(again, want, tol)
    assert ops.device_status() == 0


def test_zero_and_invalid_sequences_in_a_batch(device):
    ctx = [100, 0, 700, 64]
    pool, q, bt, cl, want, tol = decode_case(device, torch.float8_e4m3fn, torch.bfloat16, 8, 2, 128,
                                             [100, 16, 700, 64], 48)
    cl = i32([100, 0, 701 + 16, 64], device)  # none, fine but for the third: past the table
    ops.device_status()
    out = run_decode(pool, q, bt[:, :44].contiguous(), cl, [704], 2)
    assert ops.device_status() == _lib.FA_DEVERR_CONTEXT
    assert not out[1].any() and not out[2].any()
    for r in (0, 3):
        assert_close(out[r:r + 1], want[r:r + 1], tol[r:r + 1])
    out = run_decode(pool, q, bt, i32([0, -5, 0, 0], device), ctx, 2)
    assert ops.device_status() == _lib.FA_DEVERR_CONTEXT
    assert not out.any()


def test_offsets_past_32_bits(device):
    # Slabs of more than 2^32 bytes, the batch's blocks at both ends.
    H, d, nb = 8, 128, (1 << 32) // (8 * 16 * 128) + 5000
    kc = torch.zeros((nb, H, 16, d), dtype=torch.int8, device=device)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.zeros((nb, H), device=device) for _ in "kv")
    g = gen_of(device, 49)
    ctx, ids = [60, 75], [[3, nb - 1, 0, nb - 7, 0], [nb - 2, 1, nb - 3, 5, nb - 4]]
    bt = np.array(ids, np.int32)
    key, value = (torch.randn((135, H, d), device=device, generator=g).to(torch.bfloat16) for _ in "kv")
    ops.paged_append_kv8(kc, vc, ks, vs, key, value, i32(bt, device), i32(ctx, device), i32([0, 60, 135], device))
    q = torch.randn((135, 32, d), device=device, generator=g).to(torch.bfloat16)
    small = {int(b): i for i, b in enumerate(sorted({b for r in ids for b in r}))}
    at = torch.tensor(sorted(small), device=device)
    pool = tuple(t[at] for t in (kc, vc, ks, vs))
    bt_small = np.vectorize(lambda b: small[int(b)])(bt).astype(np.int32)
    raw, sc = np.zeros(pool[0].shape, np.uint8), np.zeros(pool[2].shape, np.float32)
    append_ref(raw, sc, torch.int8, key.double().cpu().numpy(), bt_small, ctx, ctx)
    np.testing.assert_array_equal(pool[0].view(torch.uint8).cpu().numpy(), raw)
    np.testing.assert_array_equal(pool[2].cpu().numpy(), sc)
    big = (kc, vc, ks, vs)
    assert torch.equal(run_prefill(big, q, bt, ctx, ctx, H, device), run_prefill(pool, q, bt_small, ctx, ctx, H, device))
    last = q[[59, 134]].contiguous()
    assert torch.equal(run_decode(big, last, i32(bt, device), i32(ctx, device), ctx, H),
                       run_decode(pool, last, i32(bt_small, device), i32(ctx, device), ctx, H))
    assert ops.device_status() == 0


def test_a_layer_from_activations_to_answers(device):
    # qkv_rope_cache into a staging layer of one block, append, attention, o_proj, logits and their
    # log probabilities: a prompt and then a decode step, as the integration notes describe.
    from flour_b200.paged import rope_tables
    H, Hq, d, hidden, V = 2, 8, 128, 256, 1024
    g = gen_of(device, 54)
    rnd = lambda *s: torch.randn(s, device=device, generator=g)  # noqa: E731
    w = (rnd((Hq + 2 * H) * d, hidden) / 16).to(torch.bfloat16)
    wo, head = (rnd(hidden, Hq * d) / 32).to(torch.bfloat16), rnd(V, hidden).to(torch.bfloat16)
    cos, sin = rope_tables(d, 64, 10000.0, torch.bfloat16, device)
    lens = [21, 40]
    bt, nb = make_tables([c + 1 for c in lens], 16, 54)
    pool = random_pool(nb, H, 16, d, torch.float8_e4m3fn, g, device)
    ws = ops.Workspace()
    for step in range(2):
        new = lens if step == 0 else [1, 1]
        ctx = [c + step for c in lens]
        n = sum(new)
        x = rnd(n, hidden).to(torch.bfloat16)
        pos = i32(np.concatenate([np.arange(c - k, c) for c, k in zip(ctx, new)]), device)
        kst, vst = (torch.zeros((1, H, n, d), device=device, dtype=torch.bfloat16) for _ in "kv")
        q = ops.qkv_rope_cache(x, w, kst, vst, pos, torch.arange(n, dtype=torch.int32, device=device), Hq, cos, sin)
        key, value = kst[0].transpose(0, 1), vst[0].transpose(0, 1)
        before = clone(pool)
        run_append(pool, key, value, bt, ctx, new, device, one=step == 1)
        check_append(pool, before, key, value, bt, ctx, new)
        if step == 0:
            out = run_prefill(pool, q, bt, ctx, new, H, device, ws=ws)
        else:
            out = run_decode(pool, q, i32(bt, device), i32(ctx, device), ctx, H, ws)
        want, tol = attention_ref(q.double().cpu().numpy(), pool, torch.as_tensor(bt), ctx, new, 4,
                                  inv_sqrt(d), 2.0 ** -8 if step == 0 else U16)
        assert_close(out, want, tol)
        y = ops.o_proj_residual(out.reshape(n, -1), wo, x)
        logits = ops.last_token_logits(y, i32(np.concatenate([[0], np.cumsum(new)]), device), head)
        picked = logits.argmax(1).to(torch.int32)
        lp, ent, ids, top = ops.token_logprobs(logits, picked, 4)
        ref = torch.log_softmax(logits.double(), 1)
        # f32 results: 2^-24 for the subtraction of the maximum and of ln Z, sums to 2.4e-6 (see
        # test_gpu_logprobs), the entropy twice that times ln V + 2.
        assert (lp - ref.max(1).values).abs().max() < 1e-5 * logits.abs().max()
        assert torch.equal(ids[:, 0], picked) and torch.equal(top[:, 0], lp)
        assert (ent - -(ref.exp() * ref).sum(1)).abs().max() < 1e-4
    assert ops.device_status() == 0


def test_blocks_are_copied_with_their_scales(device):
    # Copy-on-write of an 8-bit block with fa_copy_blocks: slabs as bf16 of half the head_dim,
    # scales as f32 layers of one element.
    pool = random_pool(12, 2, 16, 128, torch.float8_e4m3fn, gen_of(device, 42), device)
    before = clone(pool)
    pairs = i32([[3, 7], [0, 11]], device)
    half = [c.view(torch.bfloat16) for c in pool[:2]]
    ops.copy_blocks([half[0]], [half[1]], pairs)
    ops.copy_blocks([pool[2][:, :, None, None]], [pool[3][:, :, None, None]], pairs)
    for now, was in zip(pool, before):
        now, was = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (now, was)]
        assert torch.equal(now[7], was[3]) and torch.equal(now[11], was[0])
        assert torch.equal(now[:7], was[:7])


def test_blocks_are_exported_and_imported_with_their_scales(device):
    # Bundles of an 8-bit pool of two layers: slabs as bf16 of half the head_dim, scales as f32
    # layers of one element (three heads: runs of 12 bytes).
    g = gen_of(device, 70)
    src = [random_pool(12, 3, 16, 128, torch.int8, g, device) for _ in range(2)]
    dst = [random_pool(9, 3, 16, 128, torch.int8, g, device) for _ in range(2)]
    before = [clone(p) for p in dst]
    ids, to = i32([7, 0, 11], device), i32([8, 1, 4], device)

    def views(pools):
        return (([p[0].view(torch.bfloat16) for p in pools], [p[1].view(torch.bfloat16) for p in pools]),
                ([p[2][:, :, None, None] for p in pools], [p[3][:, :, None, None] for p in pools]))

    for a, b in zip(views(src), views(dst)):
        ops.import_bundle_payload(*b, to, ops.export_bundle_payload(*a, ids))
    for s, d, was in zip(src, dst, before):
        for x, y, z in zip(s, d, was):
            assert torch.equal(y[to.long()], x[ids.long()])
            rest = [i for i in range(9) if i not in (8, 1, 4)]
            assert torch.equal(y[rest], z[rest])
    assert ops.device_status() == 0


def test_refusals(device):
    ctx = [40, 50]
    pool, q, bt, cl, _, _ = decode_case(device, torch.int8, torch.bfloat16, 8, 2, 128, ctx, 43)
    ws = ops.Workspace()
    k = torch.zeros((2, 2, 128), device=device, dtype=torch.bfloat16)
    bad = [
        lambda: ops.paged_decode_kv8(q, *pool, bt, cl, 3, 0.1, 50, ws),                       # n_rep
        lambda: ops.paged_decode_kv8(q, *pool, bt, cl, 4, 0.1, 65, ws),                       # table too short
        lambda: ops.paged_decode_kv8(q, *pool, bt, cl, 4, math.nan, 50, ws),
        lambda: ops.paged_decode_kv8(q[:, :, :64], *pool, bt, cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q.double(), *pool, bt, cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q.cpu(), *pool, bt, cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q, *pool, bt.long(), cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q, *pool, bt[:1], cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q, pool[0], pool[1], pool[2].double(), pool[3], bt, cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q, pool[0].view(torch.uint8), *pool[1:], bt, cl, 4, 0.1, 50, ws),
        lambda: ops.paged_decode_kv8(q, *pool, bt, cl, 4, 0.1, 50, ws, out=q[:1]),
        lambda: ops.paged_append_kv8(*pool, k, k[:1], bt, cl),
        lambda: ops.paged_append_kv8(*pool, k[:1], k[:1], bt, cl),
        lambda: ops.paged_append_kv8(*pool, k, k, bt, cl, i32([0, 1], device)),
        lambda: ops.paged_append_kv8(*pool, k.transpose(1, 2), k.transpose(1, 2), bt, cl),
        lambda: ops.paged_prefill_kv8(q, *pool, i32([0, 1], device), cl, bt, 4, 0.1, 1, 50, 9, ws),
        lambda: ops.paged_prefill_kv8(q, *pool, i32([0, 1, 2], device), cl, bt, 4, 0.1, 60, 50, 9, ws),
        lambda: ops.paged_prefill_kv8(q, *pool, i32([0, 0, 2], device), cl, bt, 4, 0.1, 2, 50, -1, ws),
        lambda: ops.paged_prefill_kv8(q, *pool, i32([0, 0, 2], device), cl, bt, 4, 0.1, 2, 50, 9, None),
    ]
    for call in bad:
        with pytest.raises(FlourAttnError):
            call()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
