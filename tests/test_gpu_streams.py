"""stream= of the 16/32-bit wrappers: another stream than the current one, which stands still
meanwhile. Workspaces, strided inputs' copies and outputs have to be in order on the stream given."""

import math

import numpy as np
import pytest
import torch

from flour_b200 import ops
from flour_b200.workloads import LLAMA8B, make_c3, make_decode

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def strided(t):
    wide = torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


def test_attention_and_projections_on_a_stream_of_their_own(device):
    b = make_decode(LLAMA8B, np.array([3000, 40, 2500]), torch.bfloat16, device, 91)
    p = make_c3(device, seed=92, dtype=torch.bfloat16, heads=LLAMA8B, num_seqs=8, group=4, lo=20, hi=300)
    pool, ppool = (b.k_caches[0], b.v_caches[0]), (p.k_caches[0], p.v_caches[0])
    ops.reshape_and_cache(*ppool, p.key, p.value, p.slot_mapping)
    g = torch.Generator(device=device).manual_seed(93)
    new = torch.randn((3, 8, 128), device=device, generator=g).to(torch.bfloat16)
    x = torch.randn((3, 256), device=device, generator=g).to(torch.bfloat16)
    w = (torch.randn((256, 256), device=device, generator=g) / 16).to(torch.bfloat16)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=device)

    def step(ws, q, pq, **kw):
        common = (b.block_tables, b.context_lens, 4, SCALE, b.max_context_len)
        pargs = (p.cu_seqlens_q, p.context_lens, p.block_tables, 4, SCALE, p.max_seqlen_q, p.max_context_len)
        return [ops.paged_decode_append(q, *pool, new, new, *common, ws, **kw),
                ops.paged_decode(q, *pool, *common, ws, **kw),
                ops.paged_decode_noalloc(q, *pool, *common, **kw),
                ops.paged_attention_varlen(q, *pool, cu, b.context_lens, b.block_tables, 4, SCALE, 1,
                                           b.max_context_len, ws, **kw),
                ops.paged_prefill(pq, *ppool, *pargs, ws, **kw),
                ops.last_token_logits(x, cu, w, **kw),
                ops.o_proj_residual(x, w, x, **kw),
                ops.export_bundle_payload([pool[0]], [pool[1]], b.block_tables[0, :3].contiguous(), **kw)]

    q, pq = strided(b.q), strided(p.q)
    ref = step(ops.Workspace(device), q, pq)
    side = torch.cuda.Stream()
    for junk_on in (torch.cuda.current_stream(), side):  # what fresh memory holds
        with torch.cuda.stream(junk_on):
            junk = [torch.full((32 << 20,), 0x5A, dtype=torch.uint8, device=device) for _ in range(6)]
            del junk
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(1_000_000_000)  # 0.5 s
    done.record()
    ws = ops.Workspace(device)
    got = step(ws, q, pq, stream=side) + step(ws, q, pq, stream=side)
    side.synchronize()
    assert not done.query()  # none of it waited for the current stream
    with torch.cuda.stream(side):
        for name, (a, c) in enumerate(zip(got, ref + ref)):
            assert torch.equal(a, c), name
    assert ops.device_status() == 0
