"""PARTIAL_ROPE, KV_WRITE and ATTENTION on the device against their definitions in 64 bits (attention_ref), at the sizes, masks, strides and
device-side values where they can go wrong.  Bounds are derived in attention_ref.attention_bound; codes and scales of the cache are exact."""
from __future__ import annotations

import ctypes as C
import math

import attention_ref as ref
import numpy as np
import pytest
import torch

from halo_b200 import backend as hb
from halo_b200 import capi

pytestmark = pytest.mark.gpu

KINDS = {"f32": (torch.float32, capi.T_F32), "f16": (torch.float16, capi.T_F16), "bf16": (torch.bfloat16, capi.T_BF16)}
STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a rounding


@pytest.fixture(scope="module")
def be():
    return hb.CudaBackend(0)


def check(rc):
    assert rc == 0, capi.last_error()


def stream():
    return torch.cuda.current_stream().cuda_stream


def heads(t):
    """A [tokens][heads][dim] tensor of any strides as its rows of heads."""
    return capi.Heads(t.data_ptr(), t.stride(0) * t.element_size(), t.stride(1) * t.element_size())


def dev(x):
    return torch.as_tensor(np.ascontiguousarray(x)).cuda()


class Case:
    """A cache and the rows of a call, on the host (numpy, for the reference) and on the device."""

    def __init__(self, seed, kind, dim, page, n_kv, group, q_len, kv_len, loud=1.0, spare=2):
        rng = np.random.default_rng(seed)
        self.rng, self.kind, self.dtype, self.type = rng, kind, *KINDS[kind]
        self.dim, self.page, self.n_kv, self.n_q = dim, page, n_kv, n_kv * group
        self.q_len, self.length = list(q_len), list(kv_len)
        self.start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.n_tokens = int(self.start[-1])
        need = [-(-x // page) for x in kv_len]
        self.max_pages = max(need + [1]) + 1
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages)
        table = np.full((len(kv_len), self.max_pages), -7, np.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = ids[at:at + m]
            at += m
        shape = (self.n_pages, n_kv, page, dim)
        self.cache = {"table": table}
        for name in ("k", "v"):
            byte = rng.integers(118, 124, shape[:2]).astype(np.uint8)
            x = rng.normal(size=shape) * loud / ref.scale_of(byte)[:, :, None, None]
            self.cache[name] = ref.e4m3_codes(x)
            self.cache[name + "_scale"] = byte
        # slots that hold no token hold anything, NaN among it
        for i, n in enumerate(kv_len):
            if n % page:
                p = table[i, n // page]
                self.cache["k"][p, :, n % page:] = 127
                self.cache["v"][p, :, n % page:] = 255
        self.q = (rng.normal(size=(max(self.n_tokens, 1), self.n_q, dim)) * loud).astype(np.float32)[:self.n_tokens]
        self.to_device()

    def to_device(self):
        self.q_dev = dev(self.q).to(self.dtype)
        self.q = self.q_dev.double().cpu().numpy()  # what the type holds
        self.dev = {k: dev(v) for k, v in self.cache.items()}
        self.start_dev, self.length_dev = dev(self.start), dev(np.array(self.length, np.int32))
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def kv(self, **kw):
        d = self.dev
        a = dict(k=d["k"].data_ptr(), v=d["v"].data_ptr(), k_scale=d["k_scale"].data_ptr(), v_scale=d["v_scale"].data_ptr(), table=d["table"].data_ptr(),
                 type=capi.KV_E4M3, n_pages=self.n_pages, n_kv=self.n_kv, head_dim=self.dim, page_tokens=self.page, max_pages=self.max_pages,
                 n_seq=len(self.length))
        a.update(kw)
        return capi.KvCache(**a)

    def rows(self, **kw):
        a = dict(start=self.start_dev.data_ptr(), length=self.length_dev.data_ptr(), n_tokens=self.n_tokens, max_tokens=max(self.q_len + [1]))
        a.update(kw)
        return capi.KvRows(**a)

    def call(self, out, causal=True, window=0, scale=None, **kw):
        a = dict(type=self.type, n_q=self.n_q, cache=self.kv(), rows=self.rows(), q=heads(self.q_dev), out=heads(out), causal=causal, window=window,
                 scale=self.dim ** -0.5 if scale is None else scale, status=self.status.data_ptr())
        a.update(kw)
        return capi.Attention(**a)

    def run(self, be, **kw):
        out = torch.full_like(self.q_dev, 77.0)
        check(be.lib.halo_cuda_attention(be.ctx, C.byref(self.call(out, **kw)), stream()))
        torch.cuda.synchronize()
        return out

    def compare(self, out, causal=True, window=0, scale=None, bad=0):
        s = self.dim ** -0.5 if scale is None else scale
        floor = np.zeros(self.q.shape)
        want, weight, top, count = ref.attention(self.q, self.cache, self.start, self.length, s, causal, window, np.full(self.q.shape, 77.0), floor)
        got = out.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        bound = ref.attention_bound(self.kind, self.dim, want, weight, top, count) + floor
        with np.errstate(invalid="ignore"):
            off = np.abs(got - want) / np.where(np.isnan(want), 1, bound)
        worst = np.nanmax(off, initial=0.0)
        assert worst <= 1.0, f"{worst:.3g} times the bound at {np.unravel_index(np.nanargmax(off), off.shape)}"
        assert int(self.status[0]) == bad
        return want


DECODE = [1, 15, 16, 17, 63, 64, 65, 129, 700]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,n_kv,group", [(64, 16, 2, 1), (64, 128, 1, 7), (128, 64, 2, 4), (128, 16, 3, 8), (256, 32, 2, 6), (256, 128, 1, 16), (128, 32, 1, 33)])
def test_decode(be, kind, dim, page, n_kv, group):
    c = Case(1, kind, dim, page, n_kv, group, [1] * len(DECODE), DECODE)
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 128), (256, 16)])
@pytest.mark.parametrize("length", [1000, 4097, 20000])
def test_decode_of_one_long_sequence(be, kind, dim, page, length):
    c = Case(2, kind, dim, page, 1, 5, [1], [length])
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,n_kv,group", [(64, 64, 2, 2), (128, 32, 1, 8), (256, 64, 1, 6)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_several_tokens(be, kind, dim, page, n_kv, group, window):
    c = Case(3, kind, dim, page, n_kv, group, [3, 1, 5, 2, 8, 4], [3, 1, 130, 64, 515, 333])
    c.compare(c.run(be, window=window), window=window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page,n_kv,group", [(64, 16, 1, 1), (128, 64, 2, 4), (128, 128, 1, 3), (256, 32, 1, 6)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 100), (False, 0)])
def test_prompts(be, kind, dim, page, n_kv, group, causal, window):
    c = Case(4, kind, dim, page, n_kv, group, [200, 1, 129, 33, 64], [200, 300, 129, 500, 65])
    c.compare(c.run(be, causal=causal, window=window), causal=causal, window=window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_prompt_of_several_tiles(be, kind, dim):
    c = Case(5, kind, dim, 64, 1, 2, [700], [1500])
    c.compare(c.run(be))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_len,kv_len", [([150, 40, 260], [2900, 1700, 260]), ([700], [2100])])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompts_of_many_tiles_to_a_block(be, kind, dim, q_len, kv_len):
    """More tiles of keys than the device has blocks by an order: blocks walk the ends of several units."""
    c = Case(23, kind, dim, 64, 6, 3, q_len, kv_len)
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("many", [False, True])
def test_rows_that_see_nothing(be, kind, dim, many):
    """Sequences without tokens, without rows, and with more rows than tokens (rows at negative positions)."""
    q_len = [2, 0, 40, 1, 3, 0, 2] if not many else [150, 0, 400, 1, 30, 0, 2]
    c = Case(6, kind, dim, 16, 2, 4, q_len, [0, 20, 17, 0, 1, 0, 2])
    want = c.compare(c.run(be))
    assert np.all(want[:q_len[0]] == 0)
    out = c.run(be, causal=False)
    c.compare(out, causal=False)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nothing_to_do(be, dim):
    c = Case(7, "bf16", dim, 16, 1, 2, [1], [5])
    out = torch.full_like(c.q_dev, 77.0)
    for kw in (dict(rows=c.rows(n_tokens=0)), dict(rows=c.rows(max_tokens=0)), dict(cache=c.kv(n_seq=0))):
        check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(out, **kw)), stream()))
    torch.cuda.synchronize()
    assert bool((out == 77.0).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [[1, 3, 2], [70, 200, 30]])
def test_rows_behind_the_last_sequence_and_padding_stay(be, kind, q_len):
    """Strided q and out inside wider rows; rows beyond start[n_seq]; rows of a sequence beyond max_tokens."""
    c = Case(8, kind, 128, 32, 2, 3, q_len, [90, 300, 200])
    n = c.n_tokens + 5
    wide = torch.full((n, c.n_q + 3, 128 + 8), 55.0, dtype=c.dtype, device="cuda")
    q = torch.zeros((n, c.n_q, 128 + 16), dtype=c.dtype, device="cuda")
    q[:c.n_tokens, :, :128] = c.q_dev
    out = wide[:, 1:1 + c.n_q, :128]
    check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(out, q=heads(q[:, :, :128]), rows=c.rows(n_tokens=n))), stream()))
    torch.cuda.synchronize()
    c.compare(out[:c.n_tokens].contiguous())
    out[:c.n_tokens] = 55.0
    assert bool((wide == 55.0).all())
    most = max(q_len) - 1
    check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(out, q=heads(q[:, :, :128]), rows=c.rows(n_tokens=n, max_tokens=most))), stream()))
    torch.cuda.synchronize()
    left = c.start[1] + most
    assert bool((wide[left] == 55.0).all()) and not bool((wide[left - 1] == 55.0).all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_operands_off_16_byte_boundaries(be, kind, rows):
    c = Case(9, kind, 128, 16, 1, 5, [rows, rows], [rows + 100, rows])
    flat = torch.zeros(c.q_dev.numel() + 8, dtype=c.dtype, device="cuda")
    q = flat[1:1 + c.q_dev.numel()].view(c.q_dev.shape)
    q.copy_(c.q_dev)
    out = torch.zeros_like(flat)[3:3 + c.q_dev.numel()].view(c.q_dev.shape)
    check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(out, q=heads(q))), stream()))
    torch.cuda.synchronize()
    c.compare(out.clone())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("uniform", [1, 4, 100])
def test_no_starts(be, kind, uniform):
    c = Case(10, kind, 128, 32, 2, 2, [uniform] * 3, [uniform, uniform + 77, uniform + 300])
    c.compare(c.run(be, rows=c.rows(start=None)))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 150])
def test_nan_and_infinite_neighbours(be, kind, dim, rows):
    """A NaN in a key or value reaches the rows that see it and, through a value, the dimension it is in, and no other row; q's infinities and NaN stay
    in their row."""
    c = Case(11, kind, dim, 16, 1, 3, [rows, rows], [rows + 40, rows + 40])
    at = rows + 40 - max(1, rows // 2)  # seen by the last half of the rows (by the one row there is)
    p = c.cache["table"][0, at // 16]
    c.cache["v"][p, 0, at % 16, 5] = 127
    p = c.cache["table"][1, at // 16]
    c.cache["k"][p, 0, at % 16, 2] = 255
    c.to_device()
    c.compare(c.run(be))
    if rows == 1:
        return
    q = c.q_dev.clone()
    q[3, 0, 1] = math.nan
    q[5, 1, 0] = math.inf
    c.q_dev, c.q = q, q.double().cpu().numpy()
    out = c.run(be).double().cpu().numpy()
    assert np.isnan(out[3, 0]).all() and np.isnan(out[5, 1]).all()
    out[3, 0], out[5, 1] = 0, 0
    assert np.isfinite(out[:rows // 2]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_page_numbers_out_of_range(be, kind, rows):
    c = Case(12, kind, 128, 16, 2, 4, [rows] * 4, [rows + 100] * 4)
    c.cache["table"][0, 1] = -1
    c.cache["table"][1, 0] = c.n_pages
    c.cache["table"][2, :] = 2 ** 31 - 1  # no page of it is there
    c.to_device()
    c.compare(c.run(be), bad=8)
    c.status.zero_()
    c.call(c.q_dev, status=None)
    c.run(be, status=None)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 50])
def test_scales_far_apart(be, kind, rows):
    """Pages of nearly no and of very large values side by side: what a token weighs does not depend on its value's scale."""
    c = Case(13, kind, 128, 16, 1, 4, [rows], [rows + 200])
    n = c.n_pages
    c.cache["v_scale"][:, 0] = np.where(np.arange(n) % 3 == 0, 87, np.where(np.arange(n) % 3 == 1, 127, 160))
    c.cache["k_scale"][:, 0] = np.where(np.arange(n) % 4 == 0, 100, 120)
    c.cache["v_scale"][c.cache["table"][0, 2], 0] = 0    # read as 2^-40
    c.cache["k_scale"][c.cache["table"][0, 3], 0] = 20
    c.to_device()
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("loud,scale", [(1e-3, None), (30.0, None), (1.0, 0.0), (1.0, -0.3)])
def test_flat_and_peaked_weights(be, kind, rows, loud, scale):
    c = Case(14, kind, 64, 32, 1, 4, [rows], [rows + 300], loud=loud)
    c.compare(c.run(be, scale=scale), scale=scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_a_first_token_that_takes_nearly_all_the_weight(be, kind, rows):
    """One key far above thousands of equal ones whose values are what the row's answer is made of: small weights keep their precision."""
    c = Case(15, kind, 128, 64, 1, 4, [rows], [3000])
    c.cache["k"][:] = 0x38  # 1.0
    c.cache["v"][c.cache["table"][0, 0], 0, 0] = 0
    c.q = np.full(c.q.shape, 0.0)
    c.q[..., :] = 9.0 / 128 ** 0.5 / 16
    c.cache["k"][c.cache["table"][0, 0], 0, 0] = 0x58  # 16.0
    c.cache["k_scale"][:] = 127
    c.to_device()
    c.compare(c.run(be))


@pytest.mark.parametrize("rows", [1, 90])
def test_pages_of_several_layers_in_one_block_and_far_offsets(be, rows):
    """Page strides of a gigabyte: offsets pass 32 bits, what lies between the pages is not touched."""
    page, dim, n_kv, kind = 16, 128, 2, "bf16"
    c = Case(16, kind, dim, page, n_kv, 2, [rows], [rows + 6 * page - rows])
    gap = 1 << 30
    size = (c.n_pages - 1) * gap + 2 * n_kv * page * dim
    block = torch.empty(size, dtype=torch.uint8, device="cuda")
    scales = torch.zeros((c.n_pages, 64), dtype=torch.uint8, device="cuda")
    for p in range(c.n_pages):
        for j, name in enumerate(("k", "v")):
            at = p * gap + j * n_kv * page * dim
            block[at:at + n_kv * page * dim] = c.dev[name][p].reshape(-1)
            scales[p, 8 * j:8 * j + n_kv] = c.dev[name + "_scale"][p]
    cache = c.kv(k=block.data_ptr(), v=block.data_ptr() + n_kv * page * dim, page_stride=gap, k_scale=scales.data_ptr(), v_scale=scales.data_ptr() + 8,
                 scale_stride=64)
    c.compare(c.run(be, cache=cache))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [[1, 1, 1], [2, 90, 1]])
def test_the_same_call_gives_the_same_bits(be, kind, q_len):
    c = Case(17, kind, 128, 32, 2, 4, q_len, [5000, 700, 3000])
    first = c.run(be)
    for _ in range(5):
        assert torch.equal(c.run(be), first)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [[1, 2, 1], [80, 1, 200]])
def test_two_streams(be, kind, q_len):
    cs = [Case(18 + i, kind, 128, 32, 2, 4, q_len, [2000, 700 + i, 3000]) for i in range(2)]
    want = [c.run(be) for c in cs]
    outs = [torch.zeros_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, o, s in zip(cs, outs, streams):
            check(be.lib.halo_cuda_attention(be.ctx, C.byref(c.call(o)), s.cuda_stream))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
def test_a_captured_call_follows_new_lengths(be, kind, dim, rows):
    """Lengths, starts, pages and contents are read when the graph runs."""
    c = Case(20, kind, dim, 32, 2, 4, [rows, rows], [2500, 1300])
    out = torch.zeros_like(c.q_dev)
    side = torch.cuda.Stream()
    args = c.call(out)
    check(be.lib.halo_cuda_attention(be.ctx, C.byref(args), side.cuda_stream))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        check(be.lib.halo_cuda_attention(be.ctx, C.byref(args), side.cuda_stream))
    for length in ([2500, 1300], [rows, 5], [0, 0], [1999, 1300]):
        c.length = length
        c.length_dev.copy_(dev(np.array(length, np.int32)))
        out.fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        c.compare(out)
    c.length = [2500, 1300]
    c.start = np.array([0, 1, rows + 1], np.int32)
    c.start_dev.copy_(dev(c.start))
    c.length_dev.copy_(dev(np.array(c.length, np.int32)))
    out.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    c.compare(out)


def test_a_batch_of_hundreds(be):
    rng = np.random.default_rng(3)
    kv = [int(x) for x in rng.integers(0, 200, 700)]
    c = Case(21, "bf16", 64, 16, 1, 2, [1] * 700, kv)
    c.compare(c.run(be))
    q = [int(x) for x in rng.integers(0, 4, 700)]
    q[300] = 200
    c = Case(22, "bf16", 64, 16, 1, 2, q, [max(a, b) for a, b in zip(q, kv)])
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 50])
def test_query_rows_of_any_magnitude(be, kind, dim, rows):
    """Neighbouring rows from 2^-14 to 2^12 times the ordinary size, with loudly and faintly scaled keys."""
    c = Case(24, kind, dim, 32, 2, 3, [rows] * 3, [rows + 90, rows + 20, rows + 200])
    c.q *= 2.0 ** (np.arange(c.q.shape[0] * c.n_q).reshape(c.q.shape[0], c.n_q, 1) * 5 % 27 - 14)
    c.q[0, 1] = 0
    c.cache["k_scale"][:] = c.rng.integers(108, 118, c.cache["k_scale"].shape)
    c.to_device()
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 50])
def test_shared_pages(be, kind, rows):
    """Sequences with a common beginning in the same pages, and a page that a sequence holds twice."""
    c = Case(25, kind, 128, 16, 2, 4, [rows] * 3, [rows + 64, rows + 80, rows + 48])
    t = c.cache["table"]
    t[1, :3] = t[0, :3]
    t[2, 1] = t[2, 0]
    c.to_device()
    c.compare(c.run(be))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [[1, 2, 1], [80, 1, 200]])
def test_two_graphs_replayed_at_once(be, kind, q_len):
    """Each of a stream of its own: their shares of units do not meet."""
    cs = [Case(26 + i, kind, 128, 32, 2, 4, q_len, [2000, 700 + i, 3000]) for i in range(2)]
    want = [c.run(be) for c in cs]
    outs = [torch.zeros_like(w) for w in want]
    streams, graphs = [torch.cuda.Stream() for _ in cs], [torch.cuda.CUDAGraph() for _ in cs]
    args = [c.call(o) for c, o in zip(cs, outs)]
    for a, s, g in zip(args, streams, graphs):
        check(be.lib.halo_cuda_attention(be.ctx, C.byref(a), s.cuda_stream))
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            check(be.lib.halo_cuda_attention(be.ctx, C.byref(a), s.cuda_stream))
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


# ---- KV_WRITE --------------------------------------------------------------------------------------------------------------------------------
def write(be, c, k, v, status=None, **kw):
    a = dict(type=c.type, cache=c.kv(), rows=c.rows(), k=heads(k), v=heads(v), status=(c.status if status is None else status).data_ptr())
    a.update(kw)
    check(be.lib.halo_cuda_kv_write(be.ctx, C.byref(capi.KvWrite(**a)), stream()))
    torch.cuda.synchronize()


def same_cache(c):
    for name in ("k", "v", "k_scale", "v_scale"):
        got, want = c.dev[name].cpu().numpy(), c.cache[name]
        if name in ("k", "v"):
            nan = (got & 127 == 127) & (want & 127 == 127)  # either sign of a NaN
            assert np.array_equal(np.where(nan, 0, got), np.where(nan, 0, want)), name
        else:
            assert np.array_equal(got, want), name


def new_rows(c, by=1.0):
    loud = np.exp(c.rng.normal(size=(c.n_tokens, c.n_kv, 1)) * 2) * by
    x = [dev((c.rng.normal(size=(c.n_tokens, c.n_kv, c.dim)) * loud).astype(np.float32)).to(c.dtype) for _ in range(2)]
    return x, [t.double().cpu().numpy() for t in x]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("q_len,kv_len", [([1, 1, 1, 1, 1], [1, 16, 17, 129, 300]), ([3, 130, 0, 1, 40], [3, 200, 50, 1, 20]), ([300, 2], [301, 0])])
def test_kv_write(be, kind, dim, page, q_len, kv_len):
    c = Case(30, kind, dim, page, 2, 1, q_len, kv_len)
    for by in (1e-3, 1.0, 40.0):  # the scale stays, then grows
        (k, v), (kh, vh) = new_rows(c, by)
        assert not ref.kv_write(c.cache, kh, vh, c.start, c.length)
        write(be, c, k, v)
        same_cache(c)
        assert int(c.status[0]) == 0


def test_kv_write_of_special_values(be):
    c = Case(31, "f32", 64, 16, 1, 1, [9], [20])
    (k, v), _ = new_rows(c)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2], k[3] = math.nan, math.inf, -math.inf, 0.0
    v[:] = 0.0                       # a page of zeros: the smallest scale there is, or the one it had
    v[8, 0, 3] = 3.4e38              # beyond the largest scale: saturated
    k[8, 0, 3] = 1e-39               # subnormal
    kh, vh = k.double().cpu().numpy(), v.double().cpu().numpy()
    ref.kv_write(c.cache, kh, vh, c.start, c.length)
    write(be, c, k, v)
    same_cache(c)


def test_kv_write_boundaries_of_the_scale(be):
    """Largest magnitudes on, just under and just over 448 * 2^e."""
    tops = [f(np.float32(448.0 * 2.0 ** e)) for e in (-45, -41, -40, -39, -9, 0, 5, 79, 80) for f in (lambda x: np.nextafter(x, np.float32(0)), lambda x: x,
                                                                                                          lambda x: np.nextafter(x, np.float32(np.inf)))]
    n = len(tops)
    c = Case(32, "f32", 64, 16, 1, 1, [16] * n, [16] * n)
    rng = np.random.default_rng(5)
    x = (rng.random((16 * n, 1, 64)) * 2 - 1).astype(np.float32) * np.repeat(np.array(tops, np.float32), 16)[:, None, None]
    x[::16, 0, 0] = tops
    k = dev(x)
    kh = k.double().cpu().numpy()
    ref.kv_write(c.cache, kh, kh, c.start, c.length)
    write(be, c, k, k.clone())
    same_cache(c)


def test_kv_write_page_numbers_out_of_range(be):
    c = Case(33, "bf16", 128, 16, 2, 1, [40, 20, 1], [40, 100, 33])
    c.cache["table"][0, 1], c.cache["table"][1, 5], c.cache["table"][2, 2] = -1, c.n_pages, 2 ** 31 - 1
    c.to_device()
    (k, v), (kh, vh) = new_rows(c)
    assert ref.kv_write(c.cache, kh, vh, c.start, c.length)
    write(be, c, k, v)
    same_cache(c)
    assert int(c.status[0]) == 8


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_kv_write_of_a_fused_products_columns(be, kind):
    """k and v as columns of q|k|v rows, off 16-byte boundaries, with rows behind the last sequence; pages of two layers in one block."""
    c = Case(34, kind, 64, 32, 2, 1, [5, 33], [37, 64])
    (k, v), (kh, vh) = new_rows(c)
    n = c.n_tokens + 4
    fused = torch.full((n, 4 * 64 + 2 * 64 + 2 * 64 + 1), 3.0, dtype=c.dtype, device="cuda")
    kc, vc = (fused[:, at:at + 128].unflatten(1, (2, 64)) for at in (256, 384))
    kc[:c.n_tokens], vc[:c.n_tokens] = k, v
    page = c.n_kv * c.page * c.dim
    block = torch.full((c.n_pages, 4, page), 9, dtype=torch.uint8, device="cuda")
    block[:, 1], block[:, 2] = c.dev["k"].view(c.n_pages, page), c.dev["v"].view(c.n_pages, page)
    cache = c.kv(k=block.data_ptr() + page, v=block.data_ptr() + 2 * page, page_stride=4 * page)
    write(be, c, kc, vc, cache=cache, rows=c.rows(n_tokens=n))
    ref.kv_write(c.cache, kh, vh, c.start, c.length)
    c.dev["k"], c.dev["v"] = block[:, 1].reshape(c.dev["k"].shape), block[:, 2].reshape(c.dev["v"].shape)
    same_cache(c)
    assert bool((block[:, 0] == 9).all()) and bool((block[:, 3] == 9).all())


def test_kv_write_a_token_at_a_time_against_all_at_once(be):
    """Whole pages get the bytes that all rows at once get, but for kept rows that fall below the smallest normal code when the scale grows."""
    c = Case(35, "f32", 128, 16, 1, 1, [48], [48])
    (k, v), (kh, vh) = new_rows(c)
    one = Case(35, "f32", 128, 16, 1, 1, [48], [48])
    for t in range(48):
        one.start_dev.copy_(dev(np.array([0, 1], np.int32)))
        one.length_dev.copy_(dev(np.array([t + 1], np.int32)))
        write(be, one, k[t:t + 1], v[t:t + 1], rows=one.rows(n_tokens=1, max_tokens=1))
        ref.kv_write(one.cache, kh[t:t + 1], vh[t:t + 1], [0, 1], [t + 1])
    same_cache(one)
    write(be, c, k, v)
    for name in ("k", "v"):
        assert torch.equal(one.dev[name + "_scale"][c.cache["table"][0, :3]], c.dev[name + "_scale"][c.cache["table"][0, :3]])


def test_kv_write_captured(be):
    c = Case(36, "bf16", 128, 16, 2, 1, [1, 1], [5, 31])
    (k, v), _ = new_rows(c)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    args = capi.KvWrite(type=c.type, cache=c.kv(), rows=c.rows(), k=heads(k), v=heads(v), status=c.status.data_ptr())
    with torch.cuda.graph(graph, stream=side):
        check(be.lib.halo_cuda_kv_write(be.ctx, C.byref(args), side.cuda_stream))
    for length in ([5, 31], [6, 32], [7, 16]):
        (k2, v2), (kh, vh) = new_rows(c)
        k.copy_(k2), v.copy_(v2)
        c.length = length
        c.length_dev.copy_(dev(np.array(length, np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        ref.kv_write(c.cache, kh, vh, c.start, length)
        same_cache(c)


def test_kv_write_padded_rows_and_rows_behind_the_last_sequence(be):
    """Rows that belong to no sequence, or lie beyond max_tokens, are not written anywhere."""
    c = Case(38, "bf16", 128, 16, 2, 1, [2, 5, 1], [20, 33, 1])
    (k, v), (kh, vh) = new_rows(c)
    pad = [torch.full((6, c.n_kv, c.dim), 300.0, dtype=c.dtype, device="cuda") for _ in range(2)]
    k, v = (torch.cat([t, p]) for t, p in zip((k, v), pad))
    write(be, c, k, v, rows=c.rows(n_tokens=c.n_tokens + 6))
    ref.kv_write(c.cache, kh, vh, c.start, c.length)
    same_cache(c)


# ---- PARTIAL_ROPE ----------------------------------------------------------------------------------------------------------------------------
def rope_bound(kind, x, want, n, magnitude, interleaved):
    """cos and sin: the phase is cut to 2^-32 of a turn and rounded to fp32 (2^-24 of half a turn: 2^-24 pi), sincospif 2 ulp, times the
    magnitude: 2^-21 covers them; two products and a sum in fp32: 3 * 2^-24 of |a| + |b|.  Then the rounding to the type."""
    a = np.abs(np.asarray(x, np.float64))
    pair = np.zeros_like(a)
    i, j = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    pair[..., i] = pair[..., j] = (a[..., i] + a[..., j]) * magnitude
    tiny = 2.0 ** -25 if kind == "f16" else 0
    return pair * (2.0 ** -21 + 3 * 2.0 ** -24) * (1 + STEP[kind]) + STEP[kind] * np.abs(want) * (np.arange(a.shape[-1]) < 2 * n) + tiny


ROPES = [(24, 4, 256, 64, False, 5), (24, 4, 256, 64, True, 5), (3, 1, 64, 64, False, 37), (2, 2, 128, 128, True, 300), (5, 0, 128, 6, False, 9),
         (2, 1, 50, 34, False, 11), (2, 1, 50, 34, True, 11), (1, 1, 2, 2, True, 1), (70, 8, 128, 128, False, 3), (2, 0, 1024, 256, False, 2),
         (0, 3, 80, 40, False, 4), (130, 2, 256, 256, True, 2)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,dim,rot,interleaved,tokens", ROPES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rope(be, kind, n_q, n_kv, dim, rot, interleaved, tokens, in_place):
    dtype, kind_id = KINDS[kind]
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k = (torch.randn((tokens, n, dim), device="cuda", generator=gen).to(dtype) for n in (n_q, n_kv))
    pos = torch.randint(-100, 1 << 20, (tokens,), dtype=torch.int32, device="cuda", generator=gen)
    pos[0] = 2 ** 31 - 1
    pos[-1] = -2 ** 31 if tokens > 1 else 12345
    f = hb.rope_freqs(rot, 1e6, "linear", 4.0)
    freqs, magnitude = ref.rope_freqs(rot, 1e6, "linear", 4.0)
    x = [t.double().cpu().numpy() for t in (q, k)]
    outs = [q, k] if in_place else [torch.full_like(q, 7.0), torch.full_like(k, 7.0)]
    a = capi.Rope(type=kind_id, interleaved=interleaved, freqs=C.pointer(f), positions=pos.data_ptr(), q=heads(q), k=heads(k), q_out=heads(outs[0]),
                  k_out=heads(outs[1]), n_tokens=tokens, n_q=n_q, n_kv=n_kv, head_dim=dim)
    check(be.lib.halo_cuda_rope(be.ctx, C.byref(a), stream()))
    torch.cuda.synchronize()
    # the reference's own angles, in fp64, are off by 2^-53 of up to 2^31 radians: reduce its phases like the operator says instead
    turns = np.array(f.turns[:rot // 2], dtype=object)
    phase = np.array([[float((int(p) * int(t)) % (1 << 64)) * 2.0 ** -64 for t in turns] for p in pos.tolist()]) * 2 * np.pi
    near = np.abs(pos.cpu().numpy().astype(np.float64)) < 2 ** 21
    direct = np.outer(pos.cpu().numpy().astype(np.float64), freqs)
    assert np.all(np.abs(np.sin((direct - phase)[near] / 2)) < 1e-9)
    for got, want_in in zip(outs, x):
        if not want_in.size:
            continue
        want = rotate(want_in, phase, magnitude, interleaved)
        bound = rope_bound(kind, want_in, want, rot // 2, magnitude, interleaved)
        off = np.abs(got.double().cpu().numpy() - want)
        assert np.all(off <= bound), float((off / np.maximum(bound, 1e-300)).max())
        assert np.array_equal(got.double().cpu().numpy()[..., rot:], want_in[..., rot:])


def rotate(x, phase, magnitude, interleaved):
    n = phase.shape[1]
    y = np.array(x)
    c, s = np.cos(phase)[:, None] * magnitude, np.sin(phase)[:, None] * magnitude
    i, j = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("scaling,kw", [("none", {}), ("base", dict(factor=4.0)), ("ramp", dict(factor=16.0, original=32768.0, fast=32.0, slow=1.0)),
                                        ("bands", dict(factor=8.0, original=8192.0, fast=4.0, slow=1.0))])
def test_rope_in_place_in_the_columns_of_a_fused_product(be, kind, scaling, kw):
    dtype, kind_id = KINDS[kind]
    tokens, n_q, n_kv, dim, rot = 19, 4, 2, 128, 64
    fused = torch.randn((tokens, n_q + 2 * n_kv, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(dtype)
    before = fused.double().cpu().numpy()
    pos = np.arange(5000, 5000 + tokens).astype(np.int32)
    pos_dev = dev(pos)
    given = {("original_context" if k == "original" else k): v for k, v in kw.items()}
    f = hb.rope_freqs(rot, 1e6, scaling, **given)
    freqs, magnitude = ref.rope_freqs(rot, 1e6, scaling, **kw)
    q, k = heads(fused[:, :n_q]), heads(fused[:, n_q:n_q + n_kv])
    a = capi.Rope(type=kind_id, freqs=C.pointer(f), positions=pos_dev.data_ptr(), q=q, k=k, q_out=q, k_out=k, n_tokens=tokens, n_q=n_q, n_kv=n_kv, head_dim=dim)
    check(be.lib.halo_cuda_rope(be.ctx, C.byref(a), stream()))
    torch.cuda.synchronize()
    got = fused.double().cpu().numpy()
    want = before.copy()
    want[:, :n_q + n_kv] = ref.rope(before[:, :n_q + n_kv], pos, freqs, magnitude, False)
    bound = rope_bound(kind, before, want, rot // 2, magnitude, False)
    assert np.all(np.abs(got - want)[:, :n_q + n_kv] <= bound[:, :n_q + n_kv])
    assert np.array_equal(got[:, n_q + n_kv:], before[:, n_q + n_kv:])


# ---- together --------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_layer_from_prompt_to_decoded_tokens(be, kind):
    """Two sequences through the operators as a forward issues them, with the backend's own buffers and stream: a prompt, then tokens one at a time; fused
    q|k|v rows turned in place, written, attended."""
    dtype, kind_id = KINDS[kind]
    rng = np.random.default_rng(40)
    n_q, n_kv, dim, rot, page, n_pages, max_pages = 6, 2, 128, 64, 16, 12, 5
    size = 4 if kind == "f32" else 2
    row = (n_q + 2 * n_kv) * dim * size
    table = rng.permutation(n_pages)[:10].reshape(2, 5).astype(np.int32)
    host = {"k": np.zeros((n_pages, n_kv, page, dim), np.uint8), "v": np.zeros((n_pages, n_kv, page, dim), np.uint8),
            "k_scale": np.zeros((n_pages, n_kv), np.uint8), "v_scale": np.zeros((n_pages, n_kv), np.uint8), "table": table}
    st = be.create_stream()
    R = hb.TensorRef.of
    pools = {k: R(be.allocate(v.nbytes)) for k, v in host.items() if k != "table"}
    cache = hb.KvCache(pools["k"], pools["v"], pools["k_scale"], pools["v_scale"], R(be.import_host_readonly(table)), n_pages, n_kv, dim, page, max_pages, 2)
    fused, out = be.allocate(60 * row), be.allocate(60 * n_q * dim * size)
    pos_buf, start_buf, len_buf, status = be.allocate(60 * 4), be.allocate(12), be.allocate(8), be.allocate(4)
    f = hb.rope_freqs(rot, 1e6)
    freqs, magnitude = ref.rope_freqs(rot, 1e6)
    length = [0, 0]
    for step, q_len in enumerate([[20, 37], [1, 1], [1, 0], [0, 3], [1, 1], [9, 1]]):
        n = sum(q_len)
        x = torch.from_numpy(rng.normal(size=(n, n_q + 2 * n_kv, dim)).astype(np.float32)).to(dtype)
        length = [a + b for a, b in zip(length, q_len)]
        start = np.array([0, q_len[0], n], np.int32)
        pos = np.concatenate([np.arange(a - b, a) for a, b in zip(length, q_len)]).astype(np.int32)
        for buf, a in ((fused, x.view(torch.uint8).numpy()), (pos_buf, pos), (start_buf, start), (len_buf, np.array(length, np.int32))):
            be.upload(st, R(buf), a)
        q, k, v = (hb.HeadsRef(hb.TensorRef(fused, at * dim * size, 0, row)) for at in (0, n_q, n_q + n_kv))
        be.partial_rope(st, hb.RopeArgs(f, R(pos_buf), q, k, n_tokens=n, n_q=n_q, n_kv=n_kv, head_dim=dim, type=kind_id))
        be.kv_write(st, hb.KvWriteArgs(cache, k, v, R(start_buf), R(len_buf), n, 40, kind_id), status)
        be.attention(st, hb.AttentionArgs(cache, q, hb.HeadsRef(R(out)), R(start_buf), R(len_buf), n, 40, n_q, dim ** -0.5, type=kind_id), status)
        turned = torch.empty((n, n_q + 2 * n_kv, dim), dtype=dtype)
        got = torch.empty((n, n_q, dim), dtype=dtype)
        codes = {name: np.empty_like(host[name]) for name in pools}
        be.download(st, R(fused), turned.view(torch.uint8).numpy())
        be.download(st, R(out), got.view(torch.uint8).numpy())
        for name in pools:
            be.download(st, pools[name], codes[name])
        st.wait()
        xd, td = x.double().numpy(), turned.double().numpy()
        want = xd.copy()
        want[:, :n_q + n_kv] = ref.rope(xd[:, :n_q + n_kv], pos, freqs, magnitude, False)
        assert np.all(np.abs(td - want) <= rope_bound(kind, xd, want, rot // 2, magnitude, False) + 1e-300), step
        ref.kv_write(host, td[:, n_q:n_q + n_kv], td[:, n_q + n_kv:], start, length)  # from what the rope stored
        for name in pools:
            assert np.array_equal(codes[name], host[name]), (step, name)
        y, weight, top, count = ref.attention(td[:, :n_q], host, start, length, dim ** -0.5)
        assert np.all(np.abs(got.double().numpy() - y) <= ref.attention_bound(kind, dim, y, weight, top, count)), step
