"""The 8-bit cache and log-probability entry points refuse bad arguments on the host, before any
launch; the plain forms used by the GPU tests hold their own definition."""

import ctypes
import weakref

import numpy as np
import pytest
import torch

import _kv8
from flour_b200 import FlourAttnError, _lib, ops
from flour_b200._lib import FaKv8Layer, lib

P = ctypes.c_void_p
FAKE = P(0x10000)


def layer8(nb=8, kvh=2, bs=16, d=64, dt=_lib.FA_KV8_E4M3, k=0x1000, v=0x2000, ks=0x3000, vs=0x4000):
    return FaKv8Layer(k, v, ks, vs, nb, kvh, bs, d, dt)


def append(ly, dtype=_lib.FA_BF16, strides=(128, 64, 128, 64), cu=FAKE, S=1, T=3, mb=4, key=FAKE, ctx=FAKE):
    return lib().fa_paged_append_kv8(ctypes.byref(ly) if ly else None, key, FAKE, dtype, *strides, cu, ctx,
                                     FAKE, mb, S, T, None)


def decode(ly, dtype=_lib.FA_BF16, q=FAKE, mb=4, S=1, heads=4, n_rep=2, mc=64, scale=0.1, ws=None, n=0):
    return lib().fa_paged_decode_kv8(ctypes.byref(ly) if ly else None, q, FAKE, dtype, FAKE, FAKE, mb, S,
                                     heads, n_rep, mc, scale, ws, n, None)


def prefill(ly, dtype=_lib.FA_BF16, cu=FAKE, S=1, heads=4, n_rep=2, T=8, mq=8, mc=64, tb=4, ws=None, n=0):
    return lib().fa_paged_prefill_kv8(ctypes.byref(ly), FAKE, FAKE, dtype, cu, FAKE, FAKE, 4, S, heads, n_rep,
                                      T, mq, mc, tb, 0.1, ws, n, None)


def test_append_refusals():
    assert append(None) == _lib.FA_EINVAL
    assert append(layer8(dt=_lib.FA_BF16)) == _lib.FA_EINVAL
    assert append(layer8(ks=0)) == _lib.FA_EINVAL
    assert append(layer8(vs=0x4002)) == _lib.FA_EINVAL
    assert append(layer8(d=257)) == _lib.FA_EUNSUPPORTED
    assert append(layer8(bs=1025)) == _lib.FA_EUNSUPPORTED
    assert append(layer8(nb=0)) == _lib.FA_EINVAL
    assert append(layer8(), dtype=16) == _lib.FA_EINVAL
    assert append(layer8(), strides=(128, 64, -1, 64)) == _lib.FA_EINVAL
    assert append(layer8(), cu=None) == _lib.FA_EINVAL            # 3 tokens of 1 sequence need cu
    assert append(layer8(), key=None) == _lib.FA_EINVAL
    assert append(layer8(), ctx=None) == _lib.FA_EINVAL
    assert append(layer8(), key=P(0x10001)) == _lib.FA_EINVAL
    assert append(layer8(), mb=0) == _lib.FA_EINVAL
    assert append(layer8(), S=-1) == _lib.FA_EINVAL
    assert append(layer8(), T=0) == _lib.FA_OK                    # nothing to do
    assert append(layer8(), S=0, T=0, cu=None) == _lib.FA_OK


def test_attention_refusals():
    assert decode(None) == _lib.FA_EINVAL
    assert decode(layer8(), heads=5) == _lib.FA_EINVAL
    assert b"n_rep" in lib().fa_last_error_message()
    assert decode(layer8(), dtype=3) == _lib.FA_EINVAL
    assert decode(layer8(), mc=65) == _lib.FA_ERANGE
    assert decode(layer8(), mc=0) == _lib.FA_ERANGE
    assert decode(layer8(), scale=float("inf")) == _lib.FA_EINVAL
    assert decode(layer8(), q=P(0x10001)) == _lib.FA_EINVAL
    assert decode(layer8(), S=65536) == _lib.FA_EUNSUPPORTED
    assert decode(layer8(), S=0) == _lib.FA_OK
    big = layer8(nb=4096, kvh=8, d=128)
    need = lib().fa_paged_decode_kv8_workspace_size(_lib.FA_BF16, 64, 32, 8, 16, 128, 4096)
    assert need > 0
    for ws, n, st in ((None, 0, _lib.FA_EINVAL), (P(0x100000), need - 1, _lib.FA_ERANGE),
                      (P(0x100010), need, _lib.FA_EINVAL)):
        assert decode(big, mb=256, S=64, heads=32, n_rep=4, mc=4096, ws=ws, n=n) == st
    assert prefill(layer8(), cu=None) == _lib.FA_EINVAL
    assert prefill(layer8(), tb=-1) == _lib.FA_EINVAL
    assert prefill(layer8(), tb=(1 << 30) + 1) == _lib.FA_EINVAL
    assert prefill(layer8(), mq=65) == _lib.FA_ERANGE
    assert prefill(layer8(), T=0) == _lib.FA_OK
    fast = layer8(d=128)
    need = lib().fa_paged_prefill_kv8_workspace_size(_lib.FA_BF16, 1, 4, 2, 16, 128, 8, 64, 8, 4)
    assert need >= 2 * 4 * 2 * 16 * 128 * 2
    assert prefill(fast, ws=None) == _lib.FA_EINVAL
    assert prefill(fast, ws=P(0x100000), n=need - 1) == _lib.FA_ERANGE


def test_workspace_sizes_follow_the_path():
    dec, pre = lib().fa_paged_decode_kv8_workspace_size, lib().fa_paged_prefill_kv8_workspace_size
    # One token each is the decode.
    assert pre(_lib.FA_F16, 64, 32, 8, 16, 128, 64, 4096, 1, 9) == dec(_lib.FA_F16, 64, 32, 8, 16, 128, 4096) > 0
    # Shapes of the generic kernel need none.
    assert dec(_lib.FA_F32, 64, 32, 8, 16, 128, 4096) == 0
    assert dec(_lib.FA_BF16, 64, 32, 8, 8, 128, 4096) == 0
    assert dec(_lib.FA_BF16, 64, 32, 8, 16, 96, 4096) == 0
    assert dec(_lib.FA_BF16, 64, 32, 2, 16, 128, 4096) == 0   # n_rep 16
    assert dec(_lib.FA_BF16, 64, 30, 8, 16, 128, 4096) == 0   # not a multiple
    for bad in ((_lib.FA_F32, 1, 4, 2, 16, 128, 8, 64, 8, 4), (_lib.FA_BF16, 1, 4, 2, 16, 64, 8, 64, 8, 4),
                (_lib.FA_BF16, 1, 4, 2, 16, 128, 8, 64, 8, 0), (_lib.FA_BF16, 2049, 4, 2, 16, 128, 9000, 64, 8, 4)):
        assert pre(*bad) == 0
    # The copy grows with the blocks, the parts with the query rows of a long context.
    a, b = (pre(_lib.FA_BF16, 1, 28, 4, 16, 128, 509, 30001, 509, n) for n in (1876, 3752))
    assert b - a == 2 * 1876 * 4 * 16 * 128 * 2
    assert a - 2 * 1876 * 4 * 16 * 128 * 2 > 509 * 28 * 129 * 4 * 2


def test_logprobs_refusals():
    def call(dtype=0, stride=100, R=2, V=100, ids=FAKE, lp=FAKE, k=0, ti=None, tl=None, x=FAKE):
        return lib().fa_token_logprobs(x, dtype, stride, R, V, ids, lp, None, k, ti, tl, None)

    assert call(dtype=9) == _lib.FA_EINVAL
    assert call(stride=99) == _lib.FA_EINVAL
    assert call(V=0) == _lib.FA_EINVAL
    assert call(R=-1) == _lib.FA_EINVAL
    assert call(k=33, ti=FAKE, tl=FAKE) == _lib.FA_EINVAL
    assert call(k=-1) == _lib.FA_EINVAL
    assert call(k=3, ti=FAKE) == _lib.FA_EINVAL
    assert call(lp=None) == _lib.FA_EINVAL
    assert call(ids=None) == _lib.FA_EINVAL
    assert call(x=None) == _lib.FA_EINVAL
    assert call(x=P(0x10002)) == _lib.FA_EINVAL
    assert call(R=0) == _lib.FA_OK


def test_a_workspace_serves_8_bit_calls_or_the_others():
    ws = ops.Workspace()
    ws.claim(True)
    ws.claim(True)
    with pytest.raises(FlourAttnError):
        ws.claim(False)
    with pytest.raises(FlourAttnError):
        ops._ws_args(ws, 256)


def test_a_workspace_keeps_outgrown_buffers_that_graphs_hold(monkeypatch):
    ws = ops.Workspace("cpu")
    old = weakref.ref(ws.get(100))
    ws.get(1000)
    assert old() is None                  # no graph: freed
    monkeypatch.setattr(ops, "_capturing", lambda cuda: True, raising=False)
    held = weakref.ref(ws.get(500))
    monkeypatch.undo()
    at = held().data_ptr()
    assert ws.get(1000).data_ptr() == at  # still large enough
    for n in (2000, 3000):
        ws.get(n)
        assert held() is not None and held().data_ptr() == at
    assert ws.get(10).numel() == 3000


def test_a_workspace_born_in_a_capture_belongs_to_that_graph(monkeypatch):
    # What a captured call allocates holds zeros only after a replay: every captured call clears
    # its own, and eager calls take another buffer.
    ws = ops.Workspace("cpu")
    monkeypatch.setattr(ops, "_capturing", lambda cuda: True, raising=False)
    first = ws.get(100)
    first.fill_(7)
    again = ws.get(100)
    assert not again.any()
    again.fill_(7)
    monkeypatch.undo()
    eager = ws.get(100)
    assert eager.data_ptr() not in (first.data_ptr(), again.data_ptr()) and not eager.any()
    monkeypatch.setattr(ops, "_capturing", lambda cuda: True, raising=False)
    assert ws.get(100) is eager           # large enough: the graph shares it
    assert ws.get(1000).data_ptr() != eager.data_ptr()
    monkeypatch.undo()
    assert ws.get(100) is eager


def test_cpu_tensors_are_refused():
    kc = torch.zeros((4, 2, 16, 64), dtype=torch.int8)
    sc = torch.ones((4, 2))
    with pytest.raises(FlourAttnError):
        ops.paged_decode_kv8(torch.zeros(1, 4, 64), kc, kc, sc, sc, torch.zeros((1, 4), dtype=torch.int32),
                             torch.ones(1, dtype=torch.int32), 2, 0.1, 16)
    with pytest.raises(FlourAttnError):
        ops.token_logprobs(torch.zeros(2, 10))


@pytest.mark.parametrize("fmt", _kv8.FMTS)
def test_plain_encoding_agrees_with_torch(fmt):
    x = np.concatenate([np.linspace(-_kv8.QMAX[fmt], _kv8.QMAX[fmt], 20001),
                        np.array([2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 0.0, -0.0])]).astype(np.float32)
    t = torch.from_numpy(x)
    want = t.to(fmt) if fmt == torch.float8_e4m3fn else torch.round(t).to(torch.int8)
    np.testing.assert_array_equal(_kv8.encode(x.astype(np.float64), fmt), want.view(torch.uint8).numpy())
    np.testing.assert_array_equal(_kv8.decode_bytes(want.view(torch.uint8).numpy(), fmt), want.double().numpy())


@pytest.mark.parametrize("fmt", _kv8.FMTS)
def test_plain_append_loses_at_most_one_step(fmt):
    # 16 rows one by one, each twice as loud as the last: every row is re-encoded up to 15 times.
    rng = np.random.default_rng(0)
    raw, scale = np.zeros((1, 1, 16, 32), np.uint8), np.full((1, 1), 99.0, np.float32)
    x = rng.standard_normal((16, 1, 32)) * 2.0 ** np.arange(16)[:, None, None]
    for i in range(16):
        _kv8.append_ref(raw, scale, fmt, x[i:i + 1], np.zeros((1, 1), np.int32), [i + 1], [1])
    s = float(scale[0, 0])
    got = _kv8.decode_bytes(raw, fmt)[0, 0] * s
    err = np.abs(got - x[:, 0])
    if fmt == torch.int8:
        assert err.max() <= s
    else:  # half a step of 3 fraction bits, or of the subnormals' 2^-9, twice at most
        assert (err <= np.maximum(np.abs(x[:, 0]) * 2.0 ** -4, 2.0 ** -9 * s)).all()
