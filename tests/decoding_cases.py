"""Modules, data and error bounds of the decoding operators (rope, kv_append, paged_attention, matvec_w4), shared by their
CPU and GPU tests.  Element data travels as NumPy arrays the way MonoNNModule.run takes them (bf16 as uint16 patterns)."""
import numpy as np

from mononn_amd import bf16
from mononn_amd.hlo.builder import HloModuleBuilder
from oracle import decoding

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}   # a rounding is off by at most this, relative


def bits(values, dtype):
    return bf16.to_bits(values) if dtype == "bf16" else np.asarray(values).astype({"f16": np.float16, "f32": np.float32}[dtype])


def values(array, dtype):
    return bf16.from_bits(array).astype(np.float64) if dtype == "bf16" else np.asarray(array).astype(np.float64)


def module(build):
    """HLO text and outputs of a module whose entry computation `build(entry)` writes; it returns the results."""
    mb = HloModuleBuilder("cluster_0__decoding_operator.1")
    out = build(mb.entry)
    out = list(out) if isinstance(out, (list, tuple)) else [out]
    mb.entry.set_tuple_root(out)
    return mb.text(), [{"dtype": v.dtype, "dims": list(v.dims)} for v in out]


# ---- rope -------------------------------------------------------------------------------------------------------------
def rope_module(T, H, D, R, dtype, interleaved=False, amplitude=1.0):
    return module(lambda e: e.rope(e.parameter(dtype, (T, H, D), "x"), e.parameter("s32", (T,), "positions"), e.parameter("f32", (R // 2,), "inv_freq"),
                                   interleaved=interleaved, amplitude=amplitude))


def rotation_bound(x, R, dtype, interleaved, amplitude, want):
    """Half a step of the result, and the error of cosine and sine: the fraction of a turn is rounded to f32 (at most
    2^-26 turns off, 9.4e-8 rad), the functions are good to 2 ulp (1.2e-7), amplitude and the two products round once
    each: below 5e-7 of |a| + |b|."""
    a, b = np.abs(x[..., :R:2] if interleaved else x[..., :R // 2]), np.abs(x[..., 1:R:2] if interleaved else x[..., R // 2:R])
    both = np.zeros_like(x)
    if interleaved:
        both[..., 0:R:2] = both[..., 1:R:2] = a + b
    else:
        both[..., :R // 2] = both[..., R // 2:R] = a + b
    tiny = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}[dtype]
    return HALF_STEP[dtype] * (np.abs(want) + 1e-6 * both) + 5e-7 * abs(amplitude) * both + tiny


# ---- paged cache --------------------------------------------------------------------------------------------------------
def paged_batch(rng, new, ctx, page, width=None, spare=3, tokens=None):
    """page_table, query_start, context_len and the number of pages: every sequence's pages scattered over the pool,
    unused table entries -1."""
    B = len(new)
    used = [(c + page - 1) // page for c in ctx]
    width = width or max(1, max(used))
    pages = sum(used) + spare
    order = rng.permutation(pages)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    return table, np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.array(ctx, np.int32), pages


def append_module(T, H, D, pages, page, B, width, dtype, R=0, interleaved=False, amplitude=1.0):
    def build(e):
        cache = (pages, page, H, D)
        a = [e.parameter(dtype, (T, H, D), "k"), e.parameter(dtype, (T, H, D), "v"), e.parameter(dtype, cache, "k_cache"), e.parameter(dtype, cache, "v_cache"),
             e.parameter("s32", (B, width), "page_table"), e.parameter("s32", (B + 1,), "query_start"), e.parameter("s32", (B,), "context_len")]
        return e.kv_append(*a, inv_freq=e.parameter("f32", (R // 2,), "inv_freq") if R else None, interleaved=interleaved, amplitude=amplitude)
    return module(build)


def attention_module(T, H, HKV, D, pages, page, B, width, dtype, scale, window=0):
    def build(e):
        cache = (pages, page, HKV, D)
        return e.paged_attention(e.parameter(dtype, (T, H, D), "q"), e.parameter(dtype, cache, "k_cache"), e.parameter(dtype, cache, "v_cache"),
                                 e.parameter("s32", (B, width), "page_table"), e.parameter("s32", (B + 1,), "query_start"), e.parameter("s32", (B,), "context_len"),
                                 scale=scale, window=window)
    return module(build)


def attention_bound(want, mags, D, dtype):
    """w = weights, u = half a step.  Scores: D products added in f32, off by at most (D + 2) 2^-24 of the sum of their
    magnitudes, which moves a weight by that factor, numerator and sum (twice); exp2 and its argument: 2^-22 of it and
    of |score| more.  Every probability is rounded to the element type (u; below the normal range of f16 by 2^-25 at most) and the products are added in f32 (2^-22).  The sum of probabilities is at
    least 1.  The result is rounded once (u)."""
    u = HALF_STEP[dtype]
    ds = (D + 4) * 2.0 ** -24 * mags["scores"][..., None] + 2.0 ** -21
    under = 2.0 ** -25 if dtype == "f16" else 0.0
    return (u + 3 * ds + 2.0 ** -20) * mags["weighted"] + under * mags["plain"] + u * np.abs(want) * 1.01 + under


def split_attention_bound(want, mags, D, dtype):
    """attention_bound for probabilities that go into the second product in two values of the element type.  Scores as there.
    The leading value leaves less than 2^-7 (bf16, cut) or at most 2^-11 (f16) of a probability, and the second is that to
    half a step: 2^-9 of 2^-7 (the remainder's own leading bit counts), or 2^-11 of 2^-11.  In f16 a second value below the
    normal range is off by 2^-25 where the sum is at least 2^9.  The products are added in f32 (2^-22), likewise the sum."""
    ds = (D + 4) * 2.0 ** -24 * mags["scores"][..., None] + 2.0 ** -21
    lost, under, tiny = (2.0 ** -16, 0.0, 0.0) if dtype == "bf16" else (2.0 ** -22, 2.0 ** -34, 2.0 ** -25)
    return (3 * ds + lost + 2.0 ** -20) * mags["weighted"] + under * mags["plain"] + HALF_STEP[dtype] * np.abs(want) * 1.01 + tiny


# ---- 4-bit products -----------------------------------------------------------------------------------------------------
def w4_module(M, N, K, group, dtype, zeros):
    def build(e):
        x, w, s = e.parameter(dtype, (M, K), "x"), e.parameter("u8", (N, K // 2), "weight"), e.parameter(dtype, (N, K // group), "scales")
        return e.matvec_w4(x, w, s, e.parameter("u8", (N, K // group), "zeros") if zeros else None)
    return module(build)


def w4_bound(want, mags, K, group, dtype, zeros):
    """Half a step of the result; a group's products are exact and added in f32 (group steps at most), as is the sum of x
    that carries the zero point (offset by 128 + 8 in bf16, by at most 8 with zero points in f16), then the groups."""
    offset = 144 if dtype == "bf16" else (8 if zeros else 0)
    steps = group + K // group + 8
    return HALF_STEP[dtype] * np.abs(want) * 1.01 + steps * 2.0 ** -24 * (mags["products"] + 2 * offset * mags["ones"]) + (2.0 ** -25 if dtype == "f16" else 0.0)
