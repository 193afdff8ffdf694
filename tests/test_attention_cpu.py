"""The attention layer's operators without a device: the rotary frequencies, what the entry points refuse (they look at their arguments before
the context), and the references that the GPU tests go by, against torch's own conversions."""
from __future__ import annotations

import ctypes as C

import attention_ref as ref
import numpy as np
import pytest
import torch

from halo_b200 import backend as hb
from halo_b200 import capi

BASE = 0x10000000  # device addresses that no refused call looks behind


def last(rc: int, status: int, words: str) -> None:
    assert rc == status, (rc, capi.last_error())
    assert words in capi.last_error(), capi.last_error()


# ---- references ------------------------------------------------------------------------------------------------------------------------------
def test_e4m3_reference_matches_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(want, ref.VALUES.astype(np.float32), equal_nan=True)
    x = np.concatenate([np.random.default_rng(1).normal(size=20000) * 10.0 ** np.random.default_rng(2).integers(-4, 3, 20000),
                        (ref.POSITIVE[1:] + ref.POSITIVE[:-1]) / 2, -ref.POSITIVE, [0.0, -0.0, 448.0, 2.0 ** -10, 3 * 2.0 ** -10]]).astype(np.float32)
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.e4m3_codes(x), want)


def test_scale_is_the_smallest_power_of_two_that_fits():
    for top in (448.0, np.nextafter(np.float32(448), np.float32(500)), 1.0, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), 1e-30, 3e38, 0.0):
        e = ref.need_byte(float(top)) - 127
        assert e == 80 or top <= 448 * 2.0 ** e
        assert e == -40 or top > 448 * 2.0 ** (e - 1)


# ---- frequencies -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rot", [2, 6, 64, 128, 256])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp", "bands", "factors"])
def test_rope_freqs(rot, scaling):
    if scaling == "base" and rot == 2:
        with pytest.raises(hb.HaloError):
            hb.rope_freqs(rot, 1e6, scaling, 4.0)
        return
    factors = list(1 + np.arange(rot // 2) * 0.37) if scaling == "factors" else None
    kw = dict(factor=16.0, fast=32.0, slow=1.0)
    got = hb.rope_freqs(rot, 1e6, scaling, original_context=32768.0, pair_factors=factors, **kw)
    want, magnitude = ref.rope_freqs(rot, 1e6, scaling, original=32768.0, pair_factors=factors, **kw)
    assert got.n_pairs == rot // 2 and abs(got.magnitude - magnitude) <= 2.0 ** -23
    turns = np.array(got.turns[:rot // 2], np.float64) * 2.0 ** -64
    # both sides go through pow in 64 bits or more: a few roundings of 2^-53, of the exponent's product too (ln of the base, about 14, times one)
    assert np.allclose(turns, want / (2 * np.pi) % 1, rtol=2.0 ** -46, atol=2.0 ** -60)


def test_a_pairs_whole_turns_do_not_show():
    f = hb.rope_freqs(4, 1e4, "factors", pair_factors=[1 / 20.0, 1.0])  # 20 radians a position: three turns and a part
    assert abs(f.turns[0] * 2.0 ** -64 - (20 / (2 * np.pi)) % 1) < 2.0 ** -48


def test_rope_freqs_refuses():
    lib, f = capi.load(), capi.RopeFreqs()
    call = lambda rot, base, **kw: lib.halo_cuda_rope_freqs(rot, base, C.byref(capi.RopeScaling(**kw)), C.byref(f))  # noqa: E731
    assert lib.halo_cuda_rope_freqs(64, 1e4, None, C.byref(f)) == 0 and f.magnitude == 1.0
    last(lib.halo_cuda_rope_freqs(64, 1e4, None, None), capi.E_API, "null")
    for rot in (0, 63, 258):
        last(call(rot, 1e4), capi.E_KERNEL, "rotated elements")
    for base in (0.0, -1.0, float("inf"), float("nan")):
        last(call(64, base), capi.E_KERNEL, "base")
    last(call(64, 1e4, kind=6), capi.E_UNSUPPORTED, "kind 6")
    for factor in (0.0, -2.0, float("nan"), float("inf")):
        last(call(64, 1e4, kind=1, factor=factor), capi.E_KERNEL, "factor")
    last(call(64, 1e4, kind=3, factor=0.5, original_context=4096, fast=32, slow=1), capi.E_KERNEL, "factor")
    last(call(64, 1e4, kind=3, factor=4, original_context=0, fast=32, slow=1), capi.E_KERNEL, "limits")
    last(call(64, 1e4, kind=4, factor=4, original_context=4096, fast=1, slow=1), capi.E_KERNEL, "limits")
    last(call(64, 1e4, kind=5), capi.E_API, "pair factors")
    last(call(64, 1e4, magnitude=-1.0), capi.E_KERNEL, "magnitude")
    with pytest.raises(hb.HaloError):
        hb.rope_freqs(64, 1e4, "factors", pair_factors=[1.0] * 31)
    with pytest.raises(hb.HaloError):
        hb.rope_freqs(64, 1e4, "factors", pair_factors=[1.0] * 31 + [0.0])


# ---- refusals --------------------------------------------------------------------------------------------------------------------------------
def rope_call(**kw):
    f = capi.RopeFreqs(n_pairs=32, magnitude=1.0)
    a = dict(type=capi.T_F32, interleaved=0, freqs=C.pointer(f), positions=BASE, q=capi.Heads(BASE + (1 << 20), 0, 0), k=capi.Heads(BASE + (2 << 20), 0, 0),
             q_out=capi.Heads(BASE + (3 << 20), 0, 0), k_out=capi.Heads(BASE + (4 << 20), 0, 0), n_tokens=8, n_q=8, n_kv=2, head_dim=128)
    a.update(kw)
    return capi.load().halo_cuda_rope(None, C.byref(capi.Rope(**a)), None)


def test_rope_refuses():
    H, M = capi.Heads, 1 << 20
    last(rope_call(), capi.E_API, "null context")  # nothing wrong with the arguments
    last(capi.load().halo_cuda_rope(None, None, None), capi.E_API, "null argument")
    last(rope_call(type=2), capi.E_UNSUPPORTED, "type id 2")
    last(rope_call(freqs=None), capi.E_API, "frequencies")
    last(rope_call(freqs=C.pointer(capi.RopeFreqs(n_pairs=0))), capi.E_KERNEL, "pairs")
    last(rope_call(freqs=C.pointer(capi.RopeFreqs(n_pairs=129))), capi.E_KERNEL, "pairs")
    last(rope_call(freqs=C.pointer(capi.RopeFreqs(n_pairs=4, magnitude=float("nan")))), capi.E_KERNEL, "magnitude")
    last(rope_call(head_dim=62), capi.E_KERNEL, "62 elements")
    last(rope_call(head_dim=1026), capi.E_KERNEL, "1026 elements")
    last(rope_call(interleaved=2), capi.E_API, "interleaved")
    last(rope_call(positions=None), capi.E_KERNEL, "positions is empty")
    last(rope_call(positions=BASE + 2), capi.E_KERNEL, "positions is not")
    last(rope_call(q=H(None, 0, 0)), capi.E_KERNEL, "q is empty")
    last(rope_call(q=H(BASE + M + 2, 0, 0)), capi.E_KERNEL, "q is not 4-byte")
    last(rope_call(k=H(BASE + M, 0, 500)), capi.E_KERNEL, "head stride")
    last(rope_call(k=H(BASE + M, 600, 0)), capi.E_KERNEL, "token stride")
    last(rope_call(q=H(BASE + M, 2 ** 63, 0)), capi.E_KERNEL, "overflows")
    last(rope_call(q_out=H(BASE + M + 4, 0, 0)), capi.E_KERNEL, "q_out overlaps operand q")
    last(rope_call(q_out=H(BASE + 2 * M, 0, 0)), capi.E_KERNEL, "q_out overlaps operand k")
    last(rope_call(q_out=H(BASE, 0, 0)), capi.E_KERNEL, "q_out overlaps operand positions")
    last(rope_call(k_out=H(BASE + 3 * M, 0, 0)), capi.E_KERNEL, "overlaps operand k_out")
    # in place, and in place in the columns of a fused product
    same = dict(q_out=H(BASE + M, 0, 0), k_out=H(BASE + 2 * M, 0, 0))
    last(rope_call(**same), capi.E_API, "null context")
    fused = dict(q=H(BASE + M, 12 * 512, 0), q_out=H(BASE + M, 12 * 512, 0), k=H(BASE + M + 8 * 512, 12 * 512, 0), k_out=H(BASE + M + 8 * 512, 12 * 512, 0))
    last(rope_call(**fused), capi.E_API, "null context")
    fused["k_out"] = H(BASE + M + 7 * 512, 12 * 512, 0)
    last(rope_call(**fused), capi.E_KERNEL, "overlaps")


def cache(**kw):
    M = 1 << 20
    a = dict(k=BASE + 8 * M, v=BASE + 16 * M, k_scale=BASE + 24 * M, v_scale=BASE + 25 * M, table=BASE + 26 * M, type=capi.KV_E4M3, n_pages=20, n_kv=2,
             head_dim=128, page_tokens=32, max_pages=9, n_seq=3)
    a.update(kw)
    return capi.KvCache(**a)


def rows(**kw):
    a = dict(start=BASE + (27 << 20), length=BASE + (28 << 20), n_tokens=10, max_tokens=7)
    a.update(kw)
    return capi.KvRows(**a)


def write_call(**kw):
    a = dict(type=capi.T_F32, cache=cache(), rows=rows(), k=capi.Heads(BASE + (1 << 20), 0, 0), v=capi.Heads(BASE + (2 << 20), 0, 0))
    a.update(kw)
    return capi.load().halo_cuda_kv_write(None, C.byref(capi.KvWrite(**a)), None)


def attention_call(**kw):
    a = dict(type=capi.T_F32, n_q=8, cache=cache(), rows=rows(), q=capi.Heads(BASE + (1 << 20), 0, 0), out=capi.Heads(BASE + (2 << 20), 0, 0), causal=1,
             scale=0.1)
    a.update(kw)
    return capi.load().halo_cuda_attention(None, C.byref(capi.Attention(**a)), None)


@pytest.mark.parametrize("call", [write_call, attention_call])
def test_cache_refusals(call):
    M = 1 << 20
    last(call(), capi.E_API, "null context")
    last(call(type=8), capi.E_UNSUPPORTED, "type id 8")
    for bad, status, words in [(dict(type=0), capi.E_UNSUPPORTED, "cache of type id 0"), (dict(head_dim=96), capi.E_UNSUPPORTED, "96 elements"),
                               (dict(page_tokens=48), capi.E_UNSUPPORTED, "48 tokens"), (dict(page_tokens=256), capi.E_UNSUPPORTED, "256 tokens"),
                               (dict(n_kv=0), capi.E_KERNEL, "0 kv heads"), (dict(n_pages=2 ** 31), capi.E_KERNEL, "pages"),
                               (dict(max_pages=2 ** 26), capi.E_KERNEL, "sequences of"), (dict(page_stride=8000), capi.E_KERNEL, "page stride"),
                               (dict(page_stride=8200), capi.E_KERNEL, "16-byte aligned"), (dict(page_stride=2 ** 40), capi.E_KERNEL, "page stride"),
                               (dict(k=BASE + 8 * M + 8), capi.E_KERNEL, "16-byte aligned"), (dict(scale_stride=1), capi.E_KERNEL, "scale stride"),
                               (dict(table_stride=32), capi.E_KERNEL, "table stride"), (dict(table=BASE + 26 * M + 2), capi.E_KERNEL, "4-byte aligned"),
                               (dict(table_stride=38), capi.E_KERNEL, "4-byte aligned"), (dict(v=None), capi.E_KERNEL, "missing"),
                               (dict(k_scale=None), capi.E_KERNEL, "missing"), (dict(table=None), capi.E_KERNEL, "missing")]:
        last(call(cache=cache(**bad)), status, words)
    last(call(rows=rows(length=None)), capi.E_KERNEL, "lengths are missing")
    last(call(rows=rows(length=BASE + 1)), capi.E_KERNEL, "4-byte aligned")
    last(call(rows=rows(start=BASE + 2)), capi.E_KERNEL, "4-byte aligned")
    last(call(rows=rows(start=None)), capi.E_KERNEL, "rows are not")
    last(call(rows=rows(n_tokens=2 ** 31)), capi.E_KERNEL, "rows")
    last(call(rows=rows(start=None, n_tokens=21)), capi.E_API, "null context")
    last(call(status=BASE + 3), capi.E_KERNEL, "status")


def test_kv_write_refusals():
    M, H = 1 << 20, capi.Heads
    last(capi.load().halo_cuda_kv_write(None, None, None), capi.E_API, "null argument")
    last(write_call(k=H(None, 0, 0)), capi.E_KERNEL, "k is empty")
    last(write_call(v=H(BASE + 2 * M + 2, 0, 0)), capi.E_KERNEL, "v is not 4-byte")
    last(write_call(k=H(BASE + 8 * M, 0, 0)), capi.E_KERNEL, "k cache overlaps operand k")
    last(write_call(cache=cache(v=BASE + 8 * M + 4096)), capi.E_KERNEL, "overlaps operand v cache")
    last(write_call(cache=cache(v_scale=BASE + 24 * M)), capi.E_KERNEL, "overlaps")
    last(write_call(rows=rows(length=BASE + 8 * M)), capi.E_KERNEL, "overlaps operand length")
    last(write_call(cache=cache(table=BASE + 24 * M)), capi.E_KERNEL, "overlaps operand page table")
    # k and v as columns of one fused product, and the two pools of a layer interleaved page by page
    fused = dict(k=H(BASE + M, 4 * 512, 0), v=H(BASE + M + 2 * 512, 4 * 512, 0))
    last(write_call(**fused), capi.E_API, "null context")
    page = 2 * 32 * 128
    last(write_call(cache=cache(page_stride=2 * page, v=BASE + 8 * M + page)), capi.E_API, "null context")
    last(write_call(cache=cache(page_stride=2 * page, v=BASE + 8 * M + page - 16)), capi.E_KERNEL, "overlaps")


def test_attention_refusals():
    M, H = 1 << 20, capi.Heads
    last(capi.load().halo_cuda_attention(None, None, None), capi.E_API, "null argument")
    last(attention_call(n_q=0), capi.E_KERNEL, "0 query heads")
    last(attention_call(n_q=7), capi.E_KERNEL, "7 query heads")
    last(attention_call(causal=2), capi.E_API, "causal")
    last(attention_call(causal=0, window=5), capi.E_UNSUPPORTED, "window")
    last(attention_call(scale=float("nan")), capi.E_KERNEL, "scale")
    last(attention_call(scale=float("inf")), capi.E_KERNEL, "scale")
    last(attention_call(out=H(BASE + M, 0, 0)), capi.E_KERNEL, "out overlaps operand q")
    last(attention_call(out=H(BASE + 16 * M, 0, 0)), capi.E_KERNEL, "out overlaps operand v cache")
    last(attention_call(out=H(BASE + 28 * M - 64, 0, 0)), capi.E_KERNEL, "out overlaps operand length")
    last(attention_call(out=H(BASE + 2 * M, 100, 0)), capi.E_KERNEL, "token stride")


def test_the_backends_operands_are_checked_on_the_host():
    class NoBuffer(hb.Buffer):
        def __del__(self):
            pass

    be = object.__new__(hb.CudaBackend)
    be.lib, be.ctx = capi.load(), None
    f = hb.rope_freqs(64, 1e4)
    positions, q = NoBuffer(be, BASE, 16, True), NoBuffer(be, BASE + 4096, 4 * 2 * 128 * 4, True)
    a = hb.RopeArgs(f, hb.TensorRef.of(positions), hb.HeadsRef(hb.TensorRef.of(q)), n_tokens=4, n_q=2, head_dim=128)
    with pytest.raises(hb.HaloError, match="null context"):
        be.partial_rope(hb.Stream(be, 0), a)
    a.n_tokens = 5
    with pytest.raises(hb.HaloError, match="positions needs 20 bytes"):
        be.partial_rope(hb.Stream(be, 0), a)
    a.n_tokens, a.head_dim = 4, 130
    with pytest.raises(hb.HaloError, match="q needs"):
        be.partial_rope(hb.Stream(be, 0), a)
    a.head_dim, a.q.ref.buffer.writable = 128, False
    with pytest.raises(hb.HaloError, match="read-only"):
        be.partial_rope(hb.Stream(be, 0), a)


@pytest.mark.parametrize("call", [write_call, attention_call])
def test_positions_and_sequences_stay_below_what_the_device_counts_in(call):
    last(call(cache=cache(max_pages=2 ** 25, page_tokens=64, table_stride=2 ** 27)), capi.E_KERNEL, "sequences of")
    last(call(cache=cache(n_seq=2 ** 31)), capi.E_KERNEL, "2147483648 sequences")
