"""An attention layer's way through a cache held in 8 bits, as cases to be timed and compared: rotary positions, the write of keys and
values into the cache's pages, and the attention that reads them, from one decoded token to prompts of thousands.

The cache: two pools of e4m3 codes, [page][kv head][slot][dim], a page being 16 to 128 tokens; for every (page, kv head) of either pool a
byte b that stands for the scale 2^(b - 127); and for every sequence a row of page numbers.  Element = code * scale.

`own` chooses who computes: this file, in elementary torch operations (32 bits; 64 for the angles of far positions), or halo_cuda_rope,
halo_cuda_kv_write and halo_cuda_attention through the C ABI, with device pointers on torch's current stream.
24 query heads over 4 of keys and values, 256 wide with 64 rotated dimensions and base 1e7, are the attention blocks of this repository's
benchmark model; the other layouts are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MIN_BYTE, MAX_BYTE = 127 - 40, 127 + 80  # a page's scale is a power of two between 2^-40 and 2^80
MAX_FLOPS = 1.5e12   # of one pass: the largest listed attention
MAX_BYTES = 2.6e8    # likewise
MAX_CACHE = 6.0e8    # bytes of keys and values, padded: what the plain form gathers
MAX_PAIRS = 1.4e9    # padded (query row, key) pairs: what the plain form's scores may hold


def listed() -> list[dict]:
    return [
        # four sequences decode: the smallest call, a launch's latency
        {"name": "rope_token", "op": "rope", "dtype": "f32", "tokens": 4, "n_q": 24, "n_kv": 4, "dim": 256, "rot": 64, "base": 1e7,
         "interleaved": False, "scaling": "none", "far": 32768},
        # an odd number of rows of a small model with adjacent pairs and positions scaled down
        {"name": "rope_interleaved", "op": "rope", "dtype": "f16", "tokens": 1537, "n_q": 12, "n_kv": 2, "dim": 64, "rot": 64, "base": 1e4,
         "interleaved": True, "scaling": "linear", "far": 60000},
        # a long prompt far into a context that was extended by interpolating the slow dimensions
        {"name": "rope_prompt", "op": "rope", "dtype": "bf16", "tokens": 8192, "n_q": 32, "n_kv": 8, "dim": 128, "rot": 128, "base": 1e6,
         "interleaved": False, "scaling": "ramp", "far": 1000000},
        # the keys and values of 64 decoding sequences: each in the middle of a page whose scale may have to grow
        {"name": "write_tokens", "op": "write", "dtype": "f32", "n_seq": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 17, "kv_hi": 2000, "lens": 1,
         "n_kv": 4, "dim": 256, "page": 16},
        # prompts of odd lengths, some of them behind a cached prefix
        {"name": "write_prompts", "op": "write", "dtype": "bf16", "n_seq": 5, "q_lo": 900, "q_hi": 5000, "kv_lo": 900, "kv_hi": 7000, "lens": 2,
         "n_kv": 8, "dim": 128, "page": 64},
        # one sequence decodes: latency, split over its 1037 cached tokens
        {"name": "decode_one", "op": "attention", "dtype": "f32", "n_seq": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 1037, "kv_hi": 1037, "lens": 3,
         "n_q": 24, "n_kv": 4, "dim": 256, "page": 64, "causal": True, "window": 0},
        # a serving batch: 48 sequences of all lengths, small pages
        {"name": "decode_batch", "op": "attention", "dtype": "bf16", "n_seq": 48, "q_lo": 1, "q_hi": 1, "kv_lo": 150, "kv_hi": 9000, "lens": 4,
         "n_q": 32, "n_kv": 8, "dim": 128, "page": 16, "causal": True, "window": 0},
        # one sequence at the end of a long context: the cache's bytes are all that counts
        {"name": "decode_long", "op": "attention", "dtype": "bf16", "n_seq": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 131071, "kv_hi": 131071, "lens": 5,
         "n_q": 32, "n_kv": 8, "dim": 128, "page": 128, "causal": True, "window": 0},
        # speculative verify: 12 sequences of four draft tokens
        {"name": "verify", "op": "attention", "dtype": "f32", "n_seq": 12, "q_lo": 4, "q_hi": 4, "kv_lo": 1500, "kv_hi": 6000, "lens": 6,
         "n_q": 24, "n_kv": 4, "dim": 256, "page": 32, "causal": True, "window": 0},
        # a batch of whole prompts of odd lengths
        {"name": "prompts", "op": "attention", "dtype": "bf16", "n_seq": 7, "q_lo": 333, "q_hi": 3600, "kv_lo": 333, "kv_hi": 3600, "lens": 7,
         "n_q": 32, "n_kv": 8, "dim": 128, "page": 64, "causal": True, "window": 0},
        # prompts through a sliding window, a key head for every query head
        {"name": "prompts_window", "op": "attention", "dtype": "f16", "n_seq": 3, "q_lo": 1500, "q_hi": 4000, "kv_lo": 1500, "kv_hi": 4000, "lens": 8,
         "n_q": 16, "n_kv": 16, "dim": 64, "page": 32, "causal": True, "window": 1024},
        # a chunk of a long prompt behind 28000 cached tokens: the largest pass
        {"name": "chunk_long", "op": "attention", "dtype": "bf16", "n_seq": 1, "q_lo": 2048, "q_hi": 2048, "kv_lo": 30011, "kv_hi": 30011, "lens": 9,
         "n_q": 24, "n_kv": 4, "dim": 256, "page": 64, "causal": True, "window": 0},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] > MAX_BYTES or w["flops"] > MAX_FLOPS:
            continue
        if case["op"] != "attention":
            return case
        q, kv = _lengths(case)
        pairs = len(q) * max(q) * case["n_q"] * max(kv)
        cache = 2 * len(kv) * max(kv) * case["n_kv"] * case["dim"]
        if pairs <= MAX_PAIRS and cache <= MAX_CACHE:
            return case


def _draw(rng) -> dict:
    op = rng.choices(("rope", "write", "attention"), (20, 20, 60))[0]
    dtype = rng.choice(("f32", "f16", "bf16"))
    dim = rng.choice((64, 128, 256))
    n_kv = rng.choice((1, 2, 4, 8))
    n_q = n_kv * rng.choice((1, 2, 3, 4, 6, 7, 8))
    if op == "rope":
        return {"op": op, "dtype": dtype, "tokens": _log_int(rng, 1, 8192), "n_q": n_q, "n_kv": n_kv, "dim": dim,
                "rot": rng.choice((dim, dim // 2, dim // 4)), "base": rng.choice((1e4, 5e5, 1e6, 1e7)), "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(("none", "linear", "base", "ramp", "bands")), "far": _log_int(rng, 100, 1000000)}
    page = rng.choice((16, 32, 64, 128))
    lens = rng.randrange(1 << 30)
    if op == "write":
        hi = _log_int(rng, 1, 4000)
        return {"op": op, "dtype": dtype, "n_seq": _log_int(rng, 1, 128), "q_lo": max(1, hi // rng.choice((1, 2, 8))), "q_hi": hi, "kv_lo": 1,
                "kv_hi": _log_int(rng, 1, 8000), "lens": lens, "n_kv": n_kv, "dim": dim, "page": page}
    kind = rng.choice(("decode", "decode", "verify", "prompts", "chunks", "mixed"))
    case = {"op": op, "dtype": dtype, "n_seq": _log_int(rng, 1, 64), "q_lo": 1, "q_hi": 1, "kv_lo": 1, "kv_hi": 1, "lens": lens, "n_q": n_q, "n_kv": n_kv,
            "dim": dim, "page": page, "causal": True, "window": rng.choice((0, 0, 0, 128, 1000))}
    if kind in ("decode", "verify"):
        hi = _log_int(rng, 1, 60000)
        case.update(kv_lo=max(1, hi // 50), kv_hi=hi)
        if kind == "verify":
            case.update(q_lo=2, q_hi=rng.randint(2, 8))
    elif kind == "prompts":
        hi = _log_int(rng, 16, 4000)
        case.update(n_seq=_log_int(rng, 1, 8), q_lo=max(1, hi // 20), q_hi=hi, kv_lo=1, kv_hi=1, causal=rng.random() < 0.85)
    elif kind == "chunks":
        hi = _log_int(rng, 16, 2048)
        case.update(n_seq=_log_int(rng, 1, 4), q_lo=hi, q_hi=hi, kv_lo=1000, kv_hi=_log_int(rng, 1000, 20000))
    else:  # one or two prompts among decoding sequences
        case.update(n_seq=_log_int(rng, 3, 24), q_hi=_log_int(rng, 32, 1500), kv_lo=50, kv_hi=_log_int(rng, 100, 6000), mixed=True)
    if not case["causal"]:
        case["window"] = 0
    return case


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's new tokens and its length with them."""
    rng = random.Random(case["lens"])
    q, kv = [], []
    for i in range(case["n_seq"]):
        n = _log_int(rng, case["q_lo"], case["q_hi"])
        if case.get("mixed") and i >= 2:
            n = 1
        q.append(n)
        kv.append(max(n, _log_int(rng, case["kv_lo"], case["kv_hi"])))
    return q, kv


def _pairs(case: dict) -> tuple[int, int]:
    """(query, key) pairs that a mask leaves, and cached tokens that some query sees."""
    pairs = seen = 0
    w = case["window"]
    for n, length in zip(*_lengths(case)):
        if not n:
            continue
        if not case["causal"]:
            pairs, seen = pairs + n * length, seen + length
            continue
        first = length - n  # position of the first new token
        if not w:
            pairs += n * first + n * (n + 1) // 2
            seen += length
        else:
            full = max(0, length - max(first, w - 1))  # queries that see a whole window
            short = n - full
            pairs += full * w + short * first + short * (short + 1) // 2
            seen += length - max(0, first - w + 1)
    return pairs, seen


def work(case: dict):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "rope":
        n = case["tokens"] * (case["n_q"] + case["n_kv"])
        # in place only the rotated dimensions would move; into other tensors all of them do
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    q, kv = _lengths(case)
    row = case["n_kv"] * case["dim"]
    if case["op"] == "write":
        n = sum(q)
        # rows that a page held before are read, and written where its scale grows (not counted)
        kept = sum((length - n_new) % case["page"] for n_new, length in zip(q, kv) if n_new)
        return {"bytes": 2 * row * (n * (size + 1) + kept), "flops": 2 * 2 * n * row}
    pairs, seen = _pairs(case)
    return {"bytes": 2 * size * sum(q) * case["n_q"] * case["dim"] + 2 * seen * row, "flops": 4 * pairs * case["n_q"] * case["dim"]}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------
def _scaling(case: dict):
    """The parameters of each way to stretch positions: (factor, original context, fast, slow)."""
    return {"none": (1.0, 0.0, 0.0, 0.0), "linear": (8.0, 0.0, 0.0, 0.0), "base": (4.0, 0.0, 0.0, 0.0), "ramp": (16.0, 32768.0, 32.0, 1.0),
            "bands": (8.0, 8192.0, 4.0, 1.0)}[case["scaling"]]


def _pages(gen, shape, dev):
    """Codes and scale bytes as a cache holds them: values of a unit normal distribution, a few channels of them large, in e4m3."""
    x = torch.empty(shape, dtype=torch.uint8, device=dev)
    loud = 1 + 5 * (torch.rand((1, shape[1], 1, shape[3]), device=dev, generator=gen) > 0.97)
    b = torch.randint(119, 122, shape[:2], dtype=torch.uint8, device=dev, generator=gen)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, shape[0], step):
        part = torch.randn((min(step, shape[0] - at), *shape[1:]), device=dev, generator=gen) * loud
        part = part / torch.exp2(b[at:at + step].float() - 127)[:, :, None, None]
        x[at:at + step] = part.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return x, b


def prepare(case: dict, seed: int):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype, dim, n_kv = DTYPES[case["dtype"]], case["dim"], case["n_kv"]

    def normal(*shape, by=1.0):
        return (torch.randn(shape, device=dev, generator=gen) * by).to(dtype)

    if case["op"] == "rope":
        t = case["tokens"]
        q, k = normal(t, case["n_q"], dim), normal(t, n_kv, dim)
        first = int(torch.randint(0, max(1, case["far"] - t), (1,), device=dev, generator=gen))
        pos = torch.arange(first, first + t, dtype=torch.int32, device=dev)
        return {"case": case, "q": q, "k": k, "pos": pos, "freqs": _frequencies(case, dev), "q_out": torch.empty_like(q), "k_out": torch.empty_like(k)}
    q_len, kv_len = _lengths(case)
    page, n = case["page"], sum(q_len)
    need = [-(-x // page) for x in kv_len]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, device=dev, generator=gen).to(torch.int32).tolist()
    table = torch.full((len(kv_len), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    starts = [0]
    for x in q_len:
        starts.append(starts[-1] + x)
    s = {"case": case, "table": table.to(dev), "q_start": torch.tensor(starts, dtype=torch.int32, device=dev),
         "kv_len": torch.tensor(kv_len, dtype=torch.int32, device=dev), "max_q": max(q_len)}
    s["k_pool"], s["k_byte"] = _pages(gen, (n_pages, n_kv, page, dim), dev)
    s["v_pool"], s["v_byte"] = _pages(gen, (n_pages, n_kv, page, dim), dev)
    if case["op"] == "write":
        loud = torch.exp(torch.randn((n, n_kv, 1), device=dev, generator=gen)).to(dtype)
        s["k"], s["v"] = normal(n, n_kv, dim) * loud, normal(n, n_kv, dim) * loud
    else:
        s["q"] = normal(n, case["n_q"], dim, by=1.5)
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------------------------
def _frequencies(case: dict, dev):
    """(radians per position of every pair, what cosine and sine are multiplied by), in 64 bits."""
    rot, base = case["rot"], case["base"]
    factor, original, fast, slow = _scaling(case)
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if case["scaling"] == "base":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-i / rot)
    magnitude = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "ramp":
        turns_at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(turns_at(fast)), 0), min(math.ceil(turns_at(slow)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1
    elif case["scaling"] == "bands":
        turns = original * f / (2 * math.pi)  # turns of a pair over the original context
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.to(dev), magnitude


def _rotate(x, cos, sin, rot: int, interleaved: bool):
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _rope(s):
    case = s["case"]
    f, magnitude = s["freqs"]
    angle = s["pos"].double()[:, None] * f
    cos, sin = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    return [_rotate(x, cos, sin, case["rot"], case["interleaved"]) for x in (s["q"], s["k"])]


def _store(pool, scales, x, s):
    """Rows x into their slots: every touched page's scale is the smallest power of two under which its new rows fit 448, or what the rows
    kept from before it have if that is larger; kept rows are rounded again where the scale grows."""
    page = s["case"]["page"]
    n_pages, n_kv, _, _ = pool.shape
    t = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    pos = s["kv_len"].long()[seq] - s["q_start"].long()[seq + 1] + t
    at, slot = s["table"][seq, pos // page].long(), pos % page
    x = x.float()
    top = torch.zeros((n_pages, n_kv), device=x.device).index_reduce_(0, at, x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(top)
    need = (exponent - 9 + (mantissa > 0.875).int() + 127).clamp(MIN_BYTE, MAX_BYTE)
    need = torch.where(top > 0, need, MIN_BYTE)
    first = s["kv_len"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long()  # position of each sequence's first new row
    head = s["table"].gather(1, (first // page)[:, None])[:, 0].long()
    kept = (first % page)[:, None, None, None] > torch.arange(page, device=x.device)[None, None, :, None]
    old = scales[head].int()
    need[head] = torch.where(kept[:, 0, :1, 0], need[head].maximum(old), need[head])
    before = pool[head]
    again = (before.view(torch.float8_e4m3fn).float() * torch.exp2((old - need[head]).float())[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    pool[head] = torch.where(kept, again, before)
    scales[at] = need[at].to(torch.uint8)
    codes = (x * torch.exp2(127 - need[at].float())[:, :, None]).clamp(-448, 448)
    pool[at, :, slot] = codes.to(torch.float8_e4m3fn).view(torch.uint8)


def _attention(s):
    case = s["case"]
    n_seq, page, g = len(s["kv_len"]), case["page"], case["n_q"] // case["n_kv"]

    def rows(pool, scales):  # [seq][kv head][token][dim]
        at = s["table"].clamp_min(0).long()
        x = pool[at].view(torch.float8_e4m3fn).float() * torch.exp2(scales[at].float() - 127)[..., None, None]
        return x.permute(0, 2, 1, 3, 4).flatten(2, 3)

    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    seq = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    i = t - s["q_start"].long()[seq]
    q = torch.zeros((n_seq, s["max_q"], case["n_q"], case["dim"]), device=t.device)
    q[seq, i] = s["q"].float()
    q = q.view(n_seq, s["max_q"], case["n_kv"], g, case["dim"]).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seq][kv head][g * max_q][dim]
    x = q @ rows(s["k_pool"], s["k_byte"]).transpose(2, 3)
    x *= case["dim"] ** -0.5
    length = s["kv_len"].long()[:, None, None]
    key = torch.arange(s["table"].shape[1] * page, device=t.device)[None, None, :]
    at = length - (s["q_start"][1:] - s["q_start"][:-1]).long()[:, None, None] + torch.arange(s["max_q"], device=t.device)[None, :, None]
    seen = key < length
    if case["causal"]:
        seen = seen & (key <= at)
        if case["window"]:
            seen = seen & (key > at - case["window"])
    hidden = ~seen.expand(n_seq, s["max_q"], key.shape[2])
    x = x.view(n_seq, case["n_kv"], g, s["max_q"], -1).masked_fill_(hidden[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = x.exp_()
    total = p.sum(-1, keepdim=True)
    y = (p.flatten(2, 3) @ rows(s["v_pool"], s["v_byte"])).view(*total.shape[:-1], case["dim"]) / total.clamp_min(1e-30)
    return y.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, i].to(s["q"].dtype)


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------------
_context = None


def _backend():
    """One context for the process, as a host keeps it."""
    global _context
    if _context is None:
        from halo_b200 import backend
        _context = backend.CudaBackend(0)
    return _context


def _check(rc: int) -> None:
    if rc != 0:
        from halo_b200 import backend, capi
        raise backend.HaloError(rc, capi.last_error())


def _call(s):
    """The call that goes with a state: a function, and its arguments as a C host keeps them."""
    import ctypes as C

    from halo_b200 import capi
    be, case = _backend(), s["case"]
    kind = {"f32": capi.T_F32, "f16": capi.T_F16, "bf16": capi.T_BF16}[case["dtype"]]
    heads = lambda x: capi.Heads(x.data_ptr(), 0, 0)  # noqa: E731
    if case["op"] == "rope":
        factor, original, fast, slow = _scaling(case)
        scaling = capi.RopeScaling(kind=capi.ROPE_SCALINGS[case["scaling"]], factor=factor, original_context=original, fast=fast, slow=slow)
        freqs = capi.RopeFreqs()
        _check(be.lib.halo_cuda_rope_freqs(case["rot"], case["base"], C.byref(scaling), C.byref(freqs)))
        a = capi.Rope(type=kind, interleaved=case["interleaved"], freqs=C.pointer(freqs), positions=s["pos"].data_ptr(), q=heads(s["q"]), k=heads(s["k"]),
                      q_out=heads(s["q_out"]), k_out=heads(s["k_out"]), n_tokens=case["tokens"], n_q=case["n_q"], n_kv=case["n_kv"], head_dim=case["dim"])
        return be.lib.halo_cuda_rope, a, [s["q_out"], s["k_out"]]
    cache = capi.KvCache(k=s["k_pool"].data_ptr(), v=s["v_pool"].data_ptr(), k_scale=s["k_byte"].data_ptr(), v_scale=s["v_byte"].data_ptr(),
                         table=s["table"].data_ptr(), type=capi.KV_E4M3, n_pages=s["k_pool"].shape[0], n_kv=case["n_kv"], head_dim=case["dim"],
                         page_tokens=case["page"], max_pages=s["table"].shape[1], n_seq=s["table"].shape[0])
    rows = capi.KvRows(start=s["q_start"].data_ptr(), length=s["kv_len"].data_ptr(), n_tokens=(s["q"] if "q" in s else s["k"]).shape[0], max_tokens=s["max_q"])
    if case["op"] == "write":
        a = capi.KvWrite(type=kind, cache=cache, rows=rows, k=heads(s["k"]), v=heads(s["v"]))
        return be.lib.halo_cuda_kv_write, a, _caches(s)
    a = capi.Attention(type=kind, cache=cache, rows=rows, q=heads(s["q"]), out=heads(s["out"]), n_q=case["n_q"], causal=case["causal"],
                       window=case["window"], scale=case["dim"] ** -0.5)
    return be.lib.halo_cuda_attention, a, s["out"]


def _caches(s):
    f8 = torch.float8_e4m3fn
    return {"k": s["k_pool"].view(f8), "v": s["v_pool"].view(f8), "k_scale": s["k_byte"], "v_scale": s["v_byte"]}


def run(state):
    if own:
        from ctypes import byref
        if "call" not in state:
            state["call"] = _call(state)
        fn, args, outputs = state["call"]
        be = _backend()
        _check(fn(be.ctx, byref(args), torch.cuda.current_stream().cuda_stream))
        return outputs
    op = state["case"]["op"]
    if op == "rope":
        return _rope(state)
    if op == "attention":
        return _attention(state)
    _store(state["k_pool"], state["k_byte"], state["k"], state)
    _store(state["v_pool"], state["v_byte"], state["v"], state)
    return _caches(state)


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "attention": _exact_attention}[case["op"]](case, s)


def _exact_rope(case, s):
    rot, half = case["rot"], case["rot"] // 2
    factor, original, fast, slow = _scaling(case)
    base = case["base"] * (factor ** (rot / (rot - 2)) if case["scaling"] == "base" else 1)
    freqs, magnitude = [], 1.0
    for j in range(half):
        f = math.exp(-2 * j / rot * math.log(base))
        if case["scaling"] == "linear":
            f /= factor
        if case["scaling"] == "ramp":
            magnitude = 1 + math.log(factor) / 10
            lo = max(0, math.floor(rot * math.log(original / (2 * math.pi * fast)) / math.log(base * base)))
            hi = min(rot - 1, math.ceil(rot * math.log(original / (2 * math.pi * slow)) / math.log(base * base)))
            w = min(1.0, max(0.0, (j - lo) / (hi - lo or 0.001)))
            f = w * f / factor + (1 - w) * f
        if case["scaling"] == "bands":
            length = 2 * math.pi / f
            if length > original / slow:
                f /= factor
            elif length >= original / fast:
                w = (original / length - slow) / (fast - slow)
                f = (1 - w) * f / factor + w * f
        freqs.append(f)
    angle = torch.outer(s["pos"].double(), torch.tensor(freqs, dtype=torch.float64, device=s["pos"].device))
    spin = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
    outs = []
    for x in (s["q"], s["k"]):
        y = x.double()
        part = y[..., :rot]
        pair = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * spin)
        y[..., :rot] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        outs.append(y)
    return outs


def _exact_write(case, s):
    page, starts, lens, table = case["page"], s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    out = {}
    for name in ("k", "v"):
        value = s[name + "_pool"].view(torch.float8_e4m3fn).double()
        byte = s[name + "_byte"].long()
        for i, length in enumerate(lens):
            new = s[name][starts[i]:starts[i + 1]].double()
            begin = length - new.shape[0]
            at = begin
            while at < length:
                p, end = table[i][at // page], min(length, (at // page + 1) * page)
                rows = new[at - begin:end - begin].transpose(0, 1)  # [kv head][rows][dim]
                e = torch.ceil(torch.log2(rows.abs().amax((1, 2)).clamp_min(1e-300) / 448)).clamp(-40, 80)
                kept = at % page
                if kept:
                    e = torch.maximum(e, byte[p].double() - 127)
                    value[p, :, :kept] = _e4m3(value[p, :, :kept] * torch.exp2(byte[p].double() - 127 - e)[:, None, None])
                value[p, :, kept:kept + end - at] = _e4m3(rows * torch.exp2(-e)[:, None, None])
                byte[p] = (e + 127).long()
                at = end
        out[name], out[name + "_scale"] = value, byte
    return out


def _e4m3(x):
    """The nearest of +-{0, m * 2^(e - 3)}: four significant bits, none below 2^-9, none above 448; ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp_min(-9).double())
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_attention(case, s):
    g, dim, page = case["n_q"] // case["n_kv"], case["dim"], case["page"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, length in enumerate(lens):
        lo, hi = starts[i], starts[i + 1]
        if lo == hi:
            continue
        pages = s["table"][i, :-(-length // page)].long()
        pos = torch.arange(length - (hi - lo), length, device=out.device)
        key = torch.arange(length, device=out.device)
        if case["causal"]:
            far = key[None, :] > pos[:, None]
            if case["window"]:
                far |= pos[:, None] - key[None, :] >= case["window"]
        for h in range(case["n_kv"]):
            k, v = ((s[n + "_pool"][pages, h].view(torch.float8_e4m3fn).double() * torch.exp2(s[n + "_byte"][pages, h].double() - 127)[:, None, None])
                    .reshape(-1, dim)[:length] for n in ("k", "v"))
            for j in range(h * g, h * g + g):
                x = s["q"][lo:hi, j].double() @ k.T / math.sqrt(dim)
                if case["causal"]:
                    x.masked_fill_(far, -math.inf)
                out[lo:hi, j] = torch.softmax(x, -1) @ v
    return out
