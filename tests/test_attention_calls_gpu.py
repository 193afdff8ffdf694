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
