"""token_logprobs on the GPU against 64-bit log-softmax.

Tolerances (f32 results). With D the row's spread max - min over what matters (the given token, or
88, past which e^-D is 0 in f32): x - m and the subtraction of ln Z round once each at magnitudes
up to D and ln Z: 2^-24 (D + ln V) twice. Z carries a relative error of at most 2^-22 for each
2^x, and the sums of V terms in 32-long per-thread chains of tiles, then pairwise: at most
(V / 256 + 16) roundings, of random sign; 2^-24 sqrt(V) + 2^-21 covers it. The entropy adds the
same relative error of W / Z, which is at most ln V plus a constant. A streamed row's m may lie up
to 8 below its maximum: that adds 2^-24 * 16 where a token holds less than all but e^-8 of the
probability, and ln V + 1 + |result| is counted twice below: 2 (8.4 + 1) > 8.4 + 8 + 2 from 4300
logits on, which is where rows are streamed."""

import math

import numpy as np
import pytest
import torch

from flour_b200 import FlourAttnError, _lib, ops

pytestmark = pytest.mark.gpu


def reference(x, ids, k):
    """(logprobs, entropy, top ids, top logprobs) of f64 rows, by the definition."""
    x = x.double().cpu().numpy()
    R, V = x.shape
    lp = np.full(R, -np.inf)
    ent = np.zeros(R)
    top_i, top_l = np.full((R, k), -1, np.int32), np.full((R, k), -np.inf)
    for r in range(R):
        live = np.flatnonzero(x[r] > -np.inf)
        if live.size:
            m = x[r].max()
            with np.errstate(invalid="ignore"):
                z = np.log(np.exp(x[r] - m).sum())
            p = x[r] - m - z
            ent[r] = -(np.exp(p[live]) * p[live]).sum()
            lp[r] = p[ids[r]] if ids[r] >= 0 else 0.0
            order = live[np.argsort(-x[r][live], kind="stable")][:k]
            top_i[r, :order.size], top_l[r, :order.size] = order, p[order]
        elif ids[r] < 0:
            lp[r] = 0.0
    return lp, ent, top_i, top_l


def check(x, ids, k, out=None, kinds=None):
    """kinds: the rows are repetitions of the first so many."""
    ids = np.asarray(ids, np.int32)
    lp, ent, ti, tl = out or ops.token_logprobs(x, torch.as_tensor(ids, device=x.device), k)
    n = kinds or x.shape[0]
    wlp, went, wti, wtl = [np.concatenate([w] * (x.shape[0] // n)) for w in reference(x[:n], ids[:n], k)]
    V = x.shape[1]
    rel = 2.0 ** -24 * math.sqrt(V) + 2.0 ** -21
    np.testing.assert_array_equal(ti.cpu().numpy(), wti)
    for got, want in ((lp, wlp), (tl, wtl)):
        got = got.double().cpu().numpy()
        fin = np.isfinite(want)
        np.testing.assert_array_equal(got[~fin], want[~fin])
        assert (got <= 0).all()
        assert (np.abs(got[fin] - want[fin]) <= rel + 2.0 ** -23 * (np.abs(want[fin]) + math.log(V) + 1)).all()
    got = ent.double().cpu().numpy()
    assert (np.abs(got - went) <= 2 * rel * (math.log(V) + 2) + 2.0 ** -23 * (went + 1)).all(), \
        np.abs(got - went).max()
    assert ops.device_status() == 0


def logits(R, V, dtype, device, seed, scale=3.0, pad=0, shift=0):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    flat = (torch.randn(R * (V + pad) + shift, device=device, generator=g) * scale).to(dtype)
    return flat[shift:].view(R, V + pad)[:, :V]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, V, k", [(1, 1, 1), (2, 7, 5), (3, 31, 32), (5, 257, 20), (1, 8191, 1), (4, 8193, 20),
                                     (1, 151936, 20), (9, 50257, 5), (64, 128256, 20), (700, 1003, 0), (100, 40009, 20), (1, 300001, 32),
                                     (250, 33001, 5), (400, 21000, 20), (400, 8200, 20), (650, 17001, 32),
                                     (1200, 2049, 8)])
def test_sizes(device, dtype, R, V, k):
    x = logits(R, V, dtype, device, R + V)
    ids = np.random.default_rng(V).integers(0, V, R)
    check(x, ids, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad, shift", [(1, 0), (3, 1), (0, 5), (13, 3)])
def test_strides_and_alignment(device, dtype, pad, shift):
    for R, V in ((3, 20001), (300, 999)):
        x = logits(R, V, dtype, device, 5, pad=pad, shift=shift)
        check(x, np.full(R, V - 1), 20)
        check(x, np.zeros(R, np.int32), 3)


def test_neighbours_of_a_row_do_not_leak(device):
    # NaN and +inf on both sides of each row, inside its first and last 16 bytes.
    for off in range(4):
        flat = torch.full((20000,), math.nan, device=device)
        flat[off + 10000:off + 10000 + 4999] = torch.randn(4999, device=device)
        flat[off + 9999] = math.inf
        check(flat[None, off + 10000:off + 10000 + 4999], [17], 10)


@pytest.mark.parametrize("R", [1, 40, 120, 400])
def test_ties_go_to_the_lowest_id(device, R):
    V = 40000
    check(torch.zeros((R, V), device=device), [V - 1] * R, 20)                       # all equal
    check(torch.full((R, V), torch.finfo(torch.float32).min, device=device), [5] * R, 20)
    g = torch.Generator(device=device)
    g.manual_seed(1)
    x = torch.randint(-3, 4, (R, V), device=device, generator=g).to(torch.bfloat16)  # seven values
    check(x, [3] * R, 32)
    z = torch.where(torch.rand((R, V), device=device, generator=g) < 0.5, 0.0, -0.0)  # -0 == 0
    check(z, [0] * R, 16)


@pytest.mark.parametrize("step", [1, -1])
def test_sorted_rows(device, step):
    # Ascending rows make every logit a new maximum and a new candidate.
    x = torch.arange(60000, device=device, dtype=torch.float32)[None] * (1e-3 * step)
    check(x.repeat(2, 1), [0, 59999], 20)


def test_masked_rows(device):
    V = 33000
    x = logits(8, V, torch.float32, device, 9)
    keep = torch.zeros_like(x, dtype=torch.bool)
    for r, n in enumerate([0, 1, 2, 7, 19, 20, 21, V]):
        keep[r, torch.randperm(V, device=device)[:n]] = True
    x = x.masked_fill(~keep, -math.inf)
    ids = [0] + [int(keep[r].nonzero()[0]) for r in range(1, 8)]
    check(x, ids, 20)
    check(x, [-1] * 8, 20)
    dead = [int((~keep[r]).nonzero()[0]) for r in range(7)]
    lp = ops.token_logprobs(x[:7], torch.tensor(dead, dtype=torch.int32, device=device))[0]
    assert (lp == -math.inf).all()
    check(torch.where(keep, x, torch.finfo(torch.float32).min)[1:], ids[1:], 20)  # masks of the lowest value


@pytest.mark.parametrize("R", [1, 100, 300, 1200])
def test_certain_tokens(device, R):
    # One token holds all but 2^-9 ... 2^-40 of the probability: never more than all of it.
    V, n = 20000, 8
    x = logits(n, V, torch.float32, device, 21, scale=1.0)
    at = [0, 5, 4095, 8192, 12000, 16384, 19998, 19999][: min(n, R)]
    for r, i in enumerate(at):
        x[r, i] = 16.0 + 3 * r
    reps = max(1, R // n)
    x = x[: len(at)].repeat(reps, 1)
    check(x, at * reps, 5, kinds=len(at))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [144, 288, 576, 1176])  # of 1024, 512, 256 and 128 threads
def test_rows_of_all_kinds_streamed(device, R, dtype):
    # 33001 logits: every row starts at another offset from 16 bytes.
    V, kinds, info = 33001, 12, torch.finfo(dtype)
    x = logits(kinds, V, torch.float32, device, 20)
    i = torch.arange(V, device=device)
    x[1] = -math.inf
    x[2, i != 30000] = -math.inf
    x[3, i % 1600 != 7] = -math.inf             # 21 left
    x[4, i % 2 == 0] = -math.inf
    x[5] = i * 1e-3                             # ascending: every tile holds new candidates
    x[6] = i * -1e-3
    x[7] += 1e4
    x[8] = i * 1e-2                             # and new references
    x[9] = 1.5
    x[10, i % 3 > 0] = info.min                 # masks of the lowest value
    x[11, 7], x[11, 8] = info.max, info.min
    x = x.to(dtype).repeat(R // kinds, 1)
    ids = [int((x[r] > -math.inf).nonzero()[-1]) if r != 1 else -1 for r in range(kinds)] * (R // kinds)
    check(x, ids, 20, kinds=kinds)
    bad = torch.tensor([3, 20, R - 1], device=device)
    x[bad, torch.tensor([0, 16000, V - 1], device=device)] = torch.tensor([math.nan, math.inf, math.nan],
                                                                         device=device, dtype=dtype)
    x[bad[2], :V - 1] = -math.inf
    out = ops.token_logprobs(x, torch.tensor(ids, dtype=torch.int32, device=device), 20)
    for t in (out[0], out[1], out[3]):
        assert t[bad].isnan().all()
    assert (out[2][bad] == -1).all()
    good = [r for r in range(kinds, 2 * kinds) if r != 20]
    check(x[good], [ids[r] for r in good], 20, tuple(t[good] for t in out))


def test_large_offsets_and_spreads(device):
    x = logits(4, 30000, torch.float32, device, 10)
    check(x + 1e4, [1, 2, 3, 4], 5)
    check(x - 3e4, [1, 2, 3, 4], 5)
    check(x * 1e3, [1, 2, 3, 4], 5)
    big = x.clone()
    big[:, 7] = 3e38
    big[:, 8] = -3e38
    check(big, [7, 7, 7, 7], 3)


@pytest.mark.parametrize("V", [1000, 4000, 9000, 16300, 40000])
@pytest.mark.parametrize("R", [8, 160, 1200])
def test_logits_of_any_size(device, R, V):
    # f32 rows of one value c, and of c and its neighbour, from 1e6 to 3e38 of both signs: c log2(e)
    # is then far from an f32 number, and what is left of it must not push e^(x - m) out of range.
    c = torch.logspace(6, 38, 8, dtype=torch.float64)
    c[1], c[3], c[4], c[5] = 1.581e9, -1.2e10, 1.7e9, -1.591e9
    c[6] *= -1
    x = c.float().to(device)[:, None].repeat(1, V)
    x[:, V // 2] = torch.nextafter(x[:, 0], torch.full((8,), math.inf, device=device))
    x[1::4, V // 2] = x[1::4, 0]
    check(x.repeat(R // 8, 1), [V // 2, V - 1] * (R // 2), 5, kinds=8)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_nan_and_inf_rows(device, bad, dtype):
    x = logits(4, 20000, dtype, device, 11)
    x[1, 19999] = bad
    x[3] = bad
    ids = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=device)
    lp, ent, ti, tl = ops.token_logprobs(x, ids, 4)
    for r in (1, 3):
        assert lp[r].isnan() and ent[r].isnan() and tl[r].isnan().all() and (ti[r] == -1).all()
    for r in (0, 2):
        check(x[r:r + 1], [r + 1], 4, tuple(t[r:r + 1] for t in (lp, ent, ti, tl)))


def test_bad_token_ids_are_reported(device):
    x = logits(3, 1000, torch.float32, device, 12)
    ids = torch.tensor([1000, -2, 4], dtype=torch.int32, device=device)
    ops.device_status()
    lp = ops.token_logprobs(x, ids)[0]
    assert ops.device_status() == _lib.FA_DEVERR_TOKEN
    assert lp[:2].isnan().all() and not lp[2].isnan()


def test_without_tokens_without_rows_and_rows_past_32_bits(device):
    x = logits(2, 500, torch.float16, device, 13)
    lp, ent, ti, tl = ops.token_logprobs(x, None, 2)
    assert lp is None and ent.shape == (2,) and ti.shape == (2, 2)
    out = ops.token_logprobs(x[:0], torch.empty(0, dtype=torch.int32, device=device), 3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]
    # Two rows more than 2^32 bytes apart.
    flat = torch.empty((1 << 31) + 5000, dtype=torch.bfloat16, device=device)
    rows = flat.as_strided((2, 4000), ((1 << 31) + 1000, 1))
    rows.copy_(logits(2, 4000, torch.bfloat16, device, 14))
    check(rows, [3, 3999], 5)


def test_captured_and_replayed(device):
    x = logits(64, 128256, torch.float32, device, 15)
    ids = torch.randint(0, 128256, (64,), device=device, dtype=torch.int32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(x, ids, 20)
    for seed in (16, 17):
        x.copy_(logits(64, 128256, torch.float32, device, seed))
        graph.replay()
        check(x, ids.cpu().numpy(), 20, out)
    del graph


def test_refusals(device):
    x = logits(4, 100, torch.float32, device, 18)
    ids = torch.zeros(4, dtype=torch.int32, device=device)
    for call in (lambda: ops.token_logprobs(x.t(), None, 1), lambda: ops.token_logprobs(x[0], None, 1),
                 lambda: ops.token_logprobs(x, ids[:3], 1), lambda: ops.token_logprobs(x, ids.long(), 1),
                 lambda: ops.token_logprobs(x, ids, 33), lambda: ops.token_logprobs(x, ids, -1),
                 lambda: ops.token_logprobs(x.double(), ids, 1), lambda: ops.token_logprobs(x.cpu(), ids.cpu(), 1),
                 lambda: ops.token_logprobs(x, ids.cpu(), 1),
                 lambda: ops.token_logprobs(x[:1].expand(4, 100), ids, 1)):
        with pytest.raises(FlourAttnError):
            call()
    assert ops.device_status() == 0


def test_answers_of_a_step(device):
    # The step's end as a server runs it: last-token logits, then what the API answers.
    g = torch.Generator(device=device)
    g.manual_seed(19)
    hidden = torch.randn((37, 256), device=device, generator=g).to(torch.bfloat16)
    head = torch.randn((32000, 256), device=device, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, 20, 21, 37], dtype=torch.int32, device=device)
    out = ops.last_token_logits(hidden, cu, head)
    picked = out.argmax(1).to(torch.int32)
    res = ops.token_logprobs(out, picked, 5)
    check(out, picked.cpu().numpy(), 5, res)
    assert torch.equal(res[2][:, 0], picked) and torch.equal(res[3][:, 0], res[0])
