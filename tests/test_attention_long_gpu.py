"""ATTENTION over long contexts: sequences of up to a hundred million positions whose tables name a few pages again and again, so that a block
walks a long way, the cache stays small, and the answer is known from the pages alone."""
from __future__ import annotations

import ctypes as C

import attention_ref as ref
import numpy as np
import pytest
import torch

from halo_b200 import backend as hb
from halo_b200 import capi
from test_attention_gpu import Case

pytestmark = pytest.mark.gpu

KINDS = {"f32": (torch.float32, capi.T_F32), "f16": (torch.float16, capi.T_F16), "bf16": (torch.bfloat16, capi.T_BF16)}
STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a rounding
PAGE, PAGES = 128, 3


@pytest.fixture(scope="module")
def be():
    return hb.CudaBackend(0)


class Repeated:
    """One sequence of `n` positions, n_kv heads with a query head each, `rows` rows that all see the whole of it."""

    def __init__(self, seed, kind, dim, n_kv, rows, n, table=None, page=PAGE):
        rng = np.random.default_rng(seed)
        self.dtype, self.type = KINDS[kind]
        self.dim, self.n_kv, self.rows, self.n, self.page = dim, n_kv, rows, n, page
        shape = (PAGES, n_kv, page, dim)
        # values of one sign, 0.5 to 1.875: what is lost of a sum does not cancel
        self.k = rng.integers(0x20, 0x40, shape).astype(np.uint8)
        self.v = rng.integers(0x30, 0x40, shape).astype(np.uint8)
        self.table = (rng.integers(0, PAGES, -(-n // page)) if table is None else np.array(table)).astype(np.int32)
        self.dev = {name: torch.from_numpy(x).cuda() for name, x in (("k", self.k), ("v", self.v), ("table", self.table))}
        self.scales = torch.full((PAGES, n_kv), 127, dtype=torch.uint8, device="cuda")
        self.q = torch.from_numpy(rng.normal(size=(rows, n_kv, dim)).astype(np.float32)).to(self.dtype).cuda()
        self.length = torch.tensor([n], dtype=torch.int32, device="cuda")
        self.causal = 0

    def call(self, be, out, scale):
        cache = capi.KvCache(k=self.dev["k"].data_ptr(), v=self.dev["v"].data_ptr(), k_scale=self.scales.data_ptr(), v_scale=self.scales.data_ptr(),
                             table=self.dev["table"].data_ptr(), type=capi.KV_E4M3, n_pages=PAGES, n_kv=self.n_kv, head_dim=self.dim, page_tokens=self.page,
                             max_pages=len(self.table), n_seq=1)
        heads = [capi.Heads(t.data_ptr(), 0, 0) for t in (self.q, out)]
        a = capi.Attention(type=self.type, n_q=self.n_kv, cache=cache, rows=capi.KvRows(None, self.length.data_ptr(), self.rows, self.rows), q=heads[0],
                           out=heads[1], causal=self.causal, window=0, scale=scale)
        assert be.lib.halo_cuda_attention(be.ctx, C.byref(a), torch.cuda.current_stream().cuda_stream) == 0, capi.last_error()

    def time(self, be, scale):
        """Microseconds of the fastest of five calls on the device."""
        out, best = torch.empty_like(self.q), float("inf")
        for _ in range(5):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            self.call(be, out, scale)
            end.record()
            torch.cuda.synchronize()
            best = min(best, begin.elapsed_time(end) * 1e3)
        return best

    def run(self, be, scale=0.0):
        out = torch.full_like(self.q, 77.0)
        self.call(be, out, scale)
        assert be.lib.halo_cuda_stream_sync(be.ctx, torch.cuda.current_stream().cuda_stream, 0) == 0, capi.last_error()
        return out.double().cpu().numpy()

    def want(self, scale=0.0):
        """([row][kv head][dim], largest sum of |q_d k_d| * |scale|), every key of a page counted as often as the table names the page."""
        times = np.zeros((PAGES, self.page))
        np.add.at(times, self.table[:-1], 1)
        times[self.table[-1], :(self.n - 1) % self.page + 1] += 1
        k, v, q = ref.VALUES[self.k], ref.VALUES[self.v], self.q.double().cpu().numpy()
        w = np.exp(np.einsum("rhd,phtd->rhpt", q, k, optimize=True) * scale) * times
        return np.einsum("rhpt,phtd->rhd", w, v, optimize=True) / w.sum(axis=(2, 3))[..., None], np.einsum("rhd,phtd->rhpt", np.abs(q), np.abs(k), optimize=True).max() * abs(scale)


# How many products of 16 keys follow one another in the tensor cores before their sum is taken out (rows: attention_rows.cuh, 64 rows of 16-bit operands
# or 48 of fp32 at most; tiles: attention_tiles.cuh).
RUN = {("rows", "f32"): 64, ("rows", "f16"): 512, ("tiles", "f32"): 64, ("tiles", "f16"): 1024}


def few(kernel, dim):
    """(kv heads, rows) of a call of the kernel with more units than the device has blocks (three on an SM, or one): a block walks whole units."""
    return (460 if kernel == "rows" and dim < 256 else 160), (1 if kernel == "rows" else 70)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kernel,kind,n", [("rows", "f32", (1 << 18) + 5), ("rows", "f16", (1 << 23) + 70), ("tiles", "f32", (1 << 18) + 5), ("tiles", "f16", 1 << 22)])
def test_sums_of_a_long_context(be, kernel, kind, n, dim):
    """u = 2^-24.  The tensor cores cut a sum off where they add a product of 16 keys, by an ulp (2u) at most, RUN times before it is taken out; the weights'
    sum takes twice as many additions, half an ulp (u) each, in that stretch.  What was taken out is added up in fp32, u for either sum and stretch.  Joining a
    block's warps, up to 17 blocks, and the quotient: under 64 u.  Everything has one sign, so no sum on the way is larger than the last.  16-bit operands:
    a scale of zero, every weight is the same power of two and nothing but the sums can be off.  fp32: weights that differ (sums of equal ones would be exact),
    each off by what attention_ref.attention_bound says.  Then the output's own rounding."""
    run, u = RUN[kernel, kind], 2.0 ** -24
    c = Repeated(1, kind, dim, *few(kernel, dim), n)
    scale = 0.0 if kind == "f16" else 0.25 / dim
    got, (want, top) = c.run(be, scale), c.want(scale)
    keys = run // (2 if kind == "f32" else 1) * (16 if kernel == "tiles" else 64)
    weights = 0.0 if kind == "f16" else 2 * ((dim + 16) * u * top + 4 * u + 2.0 ** -22 * top) + 2.0 ** -22
    bound = 4 * run * u + 2 * (n / keys + 1) * u + 64 * u + weights + STEP[kind]
    off = np.abs(got / want - 1).max()
    print(f"{kernel} {kind} {dim}: off by {off:.3g}, bound {bound:.3g}")
    assert off <= bound


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kernel,kind", [("rows", "f32"), ("rows", "f16"), ("rows", "bf16"), ("tiles", "f32"), ("tiles", "f16"), ("tiles", "bf16")])
def test_a_maximum_that_grows_behind_sums_that_were_taken_out(be, kernel, kind, dim):
    """40960 keys of one page's and 40960 of another's, then five of a third's whose scores are about 2^10 times the others' in weight, by which everything
    before is multiplied down: the parts of the answer are of like size."""
    pages = 320
    c = Repeated(2, kind, dim, *few(kernel, dim), 2 * pages * PAGE + 5, [0] * pages + [1] * pages + [2])
    # rows of ones: a score is the mean of the key's dims times 8
    c.q = torch.ones_like(c.q)
    rng = np.random.default_rng(3)
    c.k[:] = rng.integers(0x28, 0x2A, c.k.shape)    # 0.25, 0.28: a score of about 2.1
    c.k[2] = rng.integers(0x38, 0x3A, c.k[2].shape)  # 1, 1.125: about 8.5
    c.v[1] += 8                                      # twice the first page's
    c.dev = {name: torch.from_numpy(x).cuda() for name, x in (("k", c.k), ("v", c.v), ("table", c.table))}
    scale = 8.0 / dim
    got, (want, top) = c.run(be, scale), c.want(scale)
    u, run = 2.0 ** -24, RUN[kernel, "f32" if kind == "f32" else "f16"]
    keys = run // (2 if kind == "f32" else 1) * (16 if kernel == "tiles" else 64)
    weights = 2 * ((dim + 16) * u * top + 4 * u + (2.0 ** -22 * top if kind == "f32" else 0)) + (2.0 ** -22 if kind == "f32" else 2.0 ** -11)
    bound = 4 * run * u + 4 * (c.n / keys + 1) * u + 64 * u + weights + STEP[kind]  # (a stretch's multiplication too)
    off = np.abs(got / want - 1).max()
    print(f"{kernel} {kind} {dim}: off by {off:.3g}, bound {bound:.3g}")
    assert off <= bound

@pytest.mark.parametrize("kind,rows", [("f32", 4), ("bf16", 4), ("f32", 300), ("bf16", 300)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_among_the_last_keys_costs_a_few_tiles(be, kind, rows, dim):
    """What a NaN that some rows do not see takes to come back is a look at the tiles at the edge of what they see, not at all that they see."""
    n = 60000
    c = Repeated(4, kind, dim, 8, rows, n, [0, 1] * (n // PAGE // 2) + [2])
    c.causal = 1
    clean = c.run(be, 0.5 / dim)
    last = min(rows // 2, 40)  # rows that see it, in the last page
    page, slot = c.table[(n - last) // PAGE], (n - last) % PAGE
    assert page == 2
    plain = c.time(be, 0.5 / dim)
    c.dev["v"][page, 3, slot, 5] = 127
    got, slow = c.run(be, 0.5 / dim), c.time(be, 0.5 / dim)
    nan = np.zeros(got.shape, bool)
    nan[rows - last:, 3, 5] = True
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(got[~nan], clean[~nan])
    print(f"{kind} {rows} rows of {dim}: {plain:.0f} us, with a NaN {slow:.0f}")
    assert slow < 1.5 * plain + 100


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 150])
@pytest.mark.parametrize("window", [0, 90])
def test_a_nan_beside_a_missing_page(be, kind, dim, rows, window):
    """In tiles without all of their pages NaN codes are left out of the products and put back behind them, for every row that sees them."""
    c = Case(50, kind, dim, 16, 2, 3, [rows, rows], [rows + 700, rows + 400])
    for i, at in ((0, 16 * 40 + 3), (1, 100)):
        c.cache["table"][i, at // 16 - 1] = -1
        c.cache["v"][c.cache["table"][i, at // 16], i, at % 16, 37 + i] = 255
    c.cache["v"][c.cache["table"][0, (rows + 650) // 16], 1, (rows + 650) % 16, 1] = 127  # in a tile at the edge of what some rows see, or beside it
    c.to_device()
    c.compare(c.run(be, window=window), window=window, bad=8)  # the last row sees keys from rows + 700 - 90 on: 624 to 639, of the missing page, among them


def test_a_block_may_walk_for_seconds(be):
    """A unit of 134 million positions: q of the block's next one is waited for through all of it, which takes 2.3 s, longer than a wait for
    a single step may (1.3 s)."""
    c = Repeated(5, "f16", 64, 222, 70, 1 << 27)
    got, (want, _) = c.run(be), c.want()
    run, u = RUN["tiles", "f16"], 2.0 ** -24
    assert np.abs(got / want - 1).max() <= 4 * run * u + 2 * (c.n / (run * 16) + 1) * u + 64 * u + STEP["f16"]  # as in test_sums_of_a_long_context
    assert be.lib.halo_cuda_ctx_lost(be.ctx) == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 3, 150])
def test_a_row_of_nan_that_sees_nothing_gets_zeros(be, kind, dim, rows):
    """Rows of NaN, some of which see tokens of missing pages alone: a page that is not there counts for nothing whatever it is multiplied with."""
    c = Case(51, kind, dim, 16, 2, 3, [rows] * 3, [rows, rows, rows + 300])
    c.cache["table"][0, :] = -1                  # no page of it is there
    c.cache["table"][1, :min(rows, 30) // 16 + 1] = c.n_pages  # none that its first rows see
    c.cache["table"][2, 3:11] = -5               # a whole tile of keys and parts of others
    c.to_device()
    q = c.q_dev.clone()
    q[::2, :, 5] = float("nan")
    c.q_dev, c.q = q, q.double().cpu().numpy()
    out = c.run(be)
    want = c.compare(out, bad=8)
    assert np.all(want[:rows + 1] == 0)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_among_missing_pages_costs_nothing(be, kernel, kind, dim):
    """Every tile of a long context is short of pages and has a NaN in one that is there, which all rows see."""
    n = 60000
    n_kv, rows = few(kernel, dim)
    c = Repeated(6, kind, dim, n_kv, rows, n, [0, -1, 1] * (n // 48), page=16)
    clean, plain = c.run(be, 0.5 / dim), c.time(be, 0.5 / dim)
    assert np.isfinite(clean).all()
    c.dev["v"][0, 3, 2, 5] = 255
    got, slow = c.run(be, 0.5 / dim), c.time(be, 0.5 / dim)
    nan = np.zeros(got.shape, bool)
    nan[:, 3, 5] = True
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(got[~nan], clean[~nan])
    print(f"{kernel} {kind} {dim}: {plain:.0f} us, with a NaN {slow:.0f}")
    assert slow < 1.5 * plain + 100
