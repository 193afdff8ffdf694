"""Calls of the attention layer that other tests leave out: rotations of prompts, calls without a status word, padded calls that mix prompts with
decoding sequences."""
from __future__ import annotations

import ctypes as C

import attention_ref as ref
import numpy as np
import pytest
import torch

from halo_b200 import backend as hb
from halo_b200 import capi
from test_attention_gpu import KINDS, Case, check, heads, new_rows, rope_bound, rotate, same_cache, stream, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    return hb.CudaBackend(0)


# With 2400 tokens a warp has all heads of a token, and takes 32 / (rotated elements / elements of 32 bytes) of them at a time: several turns of its loop, the
# last of them with heads for some lanes only.
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rot", [(7, 2, 256, 64), (5, 1, 128, 128), (33, 4, 64, 32), (3, 0, 256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_of_prompts(be, kind, n_q, n_kv, dim, rot, interleaved, in_place):
    dtype, kind_id = KINDS[kind]
    tokens = 2400
    gen = torch.Generator(device="cuda").manual_seed(9)
    fused = torch.randn((tokens, n_q + n_kv + 1, dim), device="cuda", generator=gen).to(dtype)  # q | k | and a column that stays
    before = fused.double().cpu().numpy()
    pos = torch.randint(-100, 1 << 20, (tokens,), dtype=torch.int32, device="cuda", generator=gen)
    f = hb.rope_freqs(rot, 1e6, "ramp", 16.0, original_context=32768.0)
    q, k = fused[:, :n_q], fused[:, n_q:n_q + n_kv]
    outs = [q, k] if in_place else [torch.full((tokens, n, dim), 7.0, dtype=dtype, device="cuda") for n in (n_q, n_kv)]
    a = capi.Rope(type=kind_id, interleaved=interleaved, freqs=C.pointer(f), positions=pos.data_ptr(), q=heads(q), k=heads(k) if n_kv else capi.Heads(),
                  q_out=heads(outs[0]), k_out=heads(outs[1]) if n_kv else capi.Heads(), n_tokens=tokens, n_q=n_q, n_kv=n_kv, head_dim=dim)
    check(be.lib.halo_cuda_rope(be.ctx, C.byref(a), stream()))
    torch.cuda.synchronize()
    turns = [int(t) for t in f.turns[:rot // 2]]
    phase = np.array([[((p * t) % (1 << 64)) * 2.0 ** -64 for t in turns] for p in pos.tolist()]) * 2 * np.pi
    for got, x in zip(outs, (before[:, :n_q], before[:, n_q:n_q + n_kv])):
        if x.shape[1]:
            want = rotate(x, phase, f.magnitude, interleaved)
            off = np.abs(got.double().cpu().numpy() - want)
            assert np.all(off <= rope_bound(kind, x, want, rot // 2, f.magnitude, interleaved))
            assert np.array_equal(got.double().cpu().numpy()[..., rot:], x[..., rot:])
    after = fused.double().cpu().numpy()
    assert np.array_equal(after[:, n_q + n_kv:] if in_place else after, before[:, n_q + n_kv:] if in_place else before)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_missing_pages_without_a_status_word(be, kind, rows):
    c = Case(60, kind, 128, 16, 2, 4, [rows] * 3, [rows + 100] * 3)
    c.cache["table"][0, 1], c.cache["table"][1, 3], c.cache["table"][2, :] = -1, c.n_pages, 2 ** 31 - 1
    c.to_device()
    c.compare(c.run(be, status=None))
    (k, v), (kh, vh) = new_rows(c)
    assert ref.kv_write(c.cache, kh, vh, c.start, c.length)
    a = capi.KvWrite(type=c.type, cache=c.kv(), rows=c.rows(), k=heads(k), v=heads(v), status=None)
    check(be.lib.halo_cuda_kv_write(be.ctx, C.byref(a), stream()))
    torch.cuda.synchronize()
    same_cache(c)
    assert int(c.status[0]) == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,n_kv,group", [(64, 16, 2, 2), (128, 64, 2, 4), (256, 32, 1, 6)])
@pytest.mark.parametrize("pad", [0, 1000])
def test_prompts_among_decoding_sequences_in_a_padded_call(be, kind, dim, page, n_kv, group, pad):
    """With pad, the call names as many rows as its sequences could have at most: the rest belongs to no sequence and stays."""
    c = Case(61, kind, dim, page, n_kv, group, [1, 1, 90, 1, 4, 0, 100, 1], [300, 20, 90, 1, 700, 50, 400, 1000])
    n = c.n_tokens + pad
    q = torch.zeros((n, c.n_q, dim), dtype=c.dtype, device="cuda")
    q[:c.n_tokens] = c.q_dev
    out = torch.full_like(q, 55.0)
    check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(out, q=heads(q), rows=c.rows(n_tokens=n))), stream()))
    torch.cuda.synchronize()
    c.compare(out[:c.n_tokens])
    assert bool((out[c.n_tokens:] == 55.0).all())
    k, v = (torch.cat([t, torch.full((pad, n_kv, dim), 300.0, dtype=c.dtype, device="cuda")]) for t in new_rows(c)[0])
    write(be, c, k, v, rows=c.rows(n_tokens=n))
    ref.kv_write(c.cache, k.double().cpu().numpy(), v.double().cpu().numpy(), c.start, c.length)
    same_cache(c)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim,gap", [(64, 16), (128, 48), (256, 16), (256, 80)])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_page_strides_that_are_no_multiple_of_a_row(be, kind, dim, gap, rows):
    c = Case(62, kind, dim, 32, 2, 4, [rows, rows], [rows + 150, rows])
    page = c.n_kv * c.page * dim
    pools = {}
    for name in ("k", "v"):
        pools[name] = torch.full((c.n_pages, page + gap), 127, dtype=torch.uint8, device="cuda")
        pools[name][:, :page] = c.dev[name].view(c.n_pages, page)
    cache = c.kv(k=pools["k"].data_ptr(), v=pools["v"].data_ptr(), page_stride=page + gap)
    c.compare(c.run(be, cache=cache))
    (k, v), (kh, vh) = new_rows(c)
    write(be, c, k, v, cache=cache)
    ref.kv_write(c.cache, kh, vh, c.start, c.length)
    for name in ("k", "v"):
        c.dev[name] = pools[name][:, :page].reshape(c.dev[name].shape)
        assert bool((pools[name][:, page:] == 127).all())
    same_cache(c)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("dim,group", [(64, 71), (128, 200), (256, 130)])
@pytest.mark.parametrize("q_len,window", [([1, 1, 1], 0), ([3, 1, 2], 0), ([5, 40, 1], 60)])
def test_many_heads_over_one(be, kind, dim, group, q_len, window):
    """A tile of packed rows has parts of a token's heads, or ends inside the next token's."""
    c = Case(63, kind, dim, 16, 1, group, q_len, [500, 40, 130])
    c.compare(c.run(be, window=window), window=window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 70])
def test_a_layers_three_calls_in_one_graph(be, kind, rows):
    """Rotation in place, write and attention of the fused rows, captured once and replayed as the context grows by them: each reads what the one in front has
    written, on a device that starts it before that one is done."""
    n_kv, group, dim, page = 2, 3, 128, 16
    c = Case(64, kind, dim, page, n_kv, group, [rows, rows], [20 + 6 * rows, 7 + 6 * rows])
    c.cache["k"][:], c.cache["v"][:], c.cache["k_scale"][:], c.cache["v_scale"][:] = 0, 0, 100, 100
    c.to_device()
    f = hb.rope_freqs(64, 1e6)
    freqs, magnitude = ref.rope_freqs(64, 1e6)
    n_q = c.n_q
    fused = torch.zeros((2 * rows, n_q + 2 * n_kv, dim), dtype=c.dtype, device="cuda")
    q, k, v = fused[:, :n_q], fused[:, n_q:n_q + n_kv], fused[:, n_q + n_kv:]
    out, pos = torch.zeros((2 * rows, n_q, dim), dtype=c.dtype, device="cuda"), torch.zeros(2 * rows, dtype=torch.int32, device="cuda")
    turn = capi.Rope(type=c.type, freqs=C.pointer(f), positions=pos.data_ptr(), q=heads(q), k=heads(k), q_out=heads(q), k_out=heads(k), n_tokens=2 * rows, n_q=n_q,
                     n_kv=n_kv, head_dim=dim)
    put = capi.KvWrite(type=c.type, cache=c.kv(), rows=c.rows(), k=heads(k), v=heads(v), status=c.status.data_ptr())
    see = c.call(out, q=heads(q))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def calls():
        check(be.lib.halo_cuda_rope(be.ctx, C.byref(turn), side.cuda_stream))
        check(be.lib.halo_cuda_kv_write(be.ctx, C.byref(put), side.cuda_stream))
        check(be.lib.halo_cuda_attention(be.ctx, C.byref(see), side.cuda_stream))

    lengths = [[20 + i * rows, 7 + i * rows] for i in range(1, 7)]
    c.length_dev.copy_(torch.tensor([0, 0], dtype=torch.int32))  # the call in front of the capture writes nothing
    torch.cuda.synchronize()
    calls()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for i, length in enumerate(lengths):
        x = torch.from_numpy(c.rng.normal(size=tuple(fused.shape)).astype(np.float32)).to(c.dtype)
        at = np.concatenate([np.arange(n - rows, n) for n in length]).astype(np.int32)
        with torch.cuda.stream(side):
            fused.copy_(x)
            pos.copy_(torch.from_numpy(at))
            c.length_dev.copy_(torch.tensor(length, dtype=torch.int32))
            graph.replay()
        torch.cuda.synchronize()
        xd, td = x.double().numpy(), fused.double().cpu().numpy()
        want = xd.copy()
        want[:, :n_q + n_kv] = ref.rope(xd[:, :n_q + n_kv], at, freqs, magnitude, False)
        assert np.all(np.abs(td - want) <= rope_bound(kind, xd, want, 32, magnitude, False) + 1e-300), i
        ref.kv_write(c.cache, td[:, n_q:n_q + n_kv], td[:, n_q + n_kv:], c.start, length)  # from what the rotation stored
        same_cache(c)
        y, weight, top, count = ref.attention(td[:, :n_q], c.cache, c.start, length, dim ** -0.5)
        assert np.all(np.abs(out.double().cpu().numpy() - y) <= ref.attention_bound(kind, dim, y, weight, top, count)), i


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 100])
def test_a_million_sequences_of_which_few_have_rows(be, kind, rows):
    """Blocks step past all that have none."""
    n = 1 << 20
    q_len, length = [0] * n, [0] * n
    for i, more in ((5, 300), (6, 0), (n // 2, 40), (n - 1, 700)):
        q_len[i], length[i] = rows, rows + more
    q_len[n // 3], length[n // 3] = 2, 20
    c = Case(65, kind, 64, 16, 1, 1, q_len, length)
    c.compare(c.run(be))
    assert be.lib.halo_cuda_stream_sync(be.ctx, stream(), 0) == 0, capi.last_error()
