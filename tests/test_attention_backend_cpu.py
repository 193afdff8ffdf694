"""The attention layer through CudaBackend, as far as it looks at operands on the host."""
from __future__ import annotations

import ctypes as C

import pytest

from halo_b200 import backend as hb
from halo_b200 import capi

BASE = 0x10000000  # device addresses that no refused call looks behind


class NoBuffer(hb.Buffer):
    def __del__(self):
        pass


def call(k_stride=0, v_stride=0, k_scale_stride=0, v_scale_stride=0, pages=3):
    """Reaches the library, which finds no context, or is refused on the way."""
    be = object.__new__(hb.CudaBackend)
    be.lib, be.ctx = capi.load(), None
    at = iter(range(BASE, 1 << 40, 1 << 24))
    ref = lambda size, stride=0: hb.TensorRef(NoBuffer(be, next(at), size, True), 0, 0, stride)  # noqa: E731
    n_kv, dim, page = 2, 64, 16
    codes = n_kv * dim * page
    cache = hb.KvCache(ref((pages - 1) * (k_stride or codes) + codes, k_stride), ref((pages - 1) * (v_stride or codes) + codes, v_stride),
                       ref((pages - 1) * (k_scale_stride or n_kv) + n_kv, k_scale_stride), ref((pages - 1) * (v_scale_stride or n_kv) + n_kv, v_scale_stride),
                       ref(8), pages, n_kv, dim, page, 2, 1)
    rows = [hb.HeadsRef(ref(4 * n_kv * dim * 4)) for _ in range(2)]
    be.kv_write(hb.Stream(be, 0), hb.KvWriteArgs(cache, *rows, length=ref(4), n_tokens=4, max_tokens=4))


def test_a_dense_pool_and_one_of_the_same_stride_in_numbers_are_alike():
    for kw in ({}, dict(k_stride=2048), dict(v_stride=2048), dict(k_scale_stride=2), dict(v_scale_stride=2), dict(k_stride=4096, v_stride=4096)):
        with pytest.raises(hb.HaloError, match="null context"):
            call(**kw)


def test_pools_of_two_strides_are_refused():
    for kw in (dict(k_stride=4096), dict(k_stride=2048, v_stride=4096), dict(v_scale_stride=3), dict(k_scale_stride=8, v_scale_stride=4)):
        with pytest.raises(hb.HaloError, match="one stride"):
            call(**kw)


def test_attention_takes_a_million_sequences():
    heads = [capi.Heads(BASE + (i << 36), 0, 0) for i in (1, 2)]
    for n_seq, status, words in ((1 << 20, capi.E_API, "null context"), ((1 << 20) + 1, capi.E_UNSUPPORTED, "1048577 sequences")):
        cache = capi.KvCache(k=BASE, v=BASE + (1 << 24), k_scale=BASE + (2 << 24), v_scale=BASE + (3 << 24), table=BASE + (4 << 36), type=capi.KV_E4M3, n_pages=2, n_kv=1,
                             head_dim=64, page_tokens=16, max_pages=1, n_seq=n_seq)
        a = capi.Attention(type=capi.T_F16, n_q=1, cache=cache, rows=capi.KvRows(BASE + (5 << 36), BASE + (6 << 36), n_seq, 1), q=heads[0], out=heads[1], causal=1, scale=1.0)
        assert capi.load().halo_cuda_attention(None, C.byref(a), None) == status
        assert words in capi.last_error()
