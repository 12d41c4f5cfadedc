"""The decoding operators on the CPU: their oracle against restatements that share nothing with it, what the compiler
refuses, how their nodes sit in a program, and the addresses their kernels touch."""
import ctypes
import json
import os

import numpy as np
import pytest

import cpu_bounds
import decoding_cases as dc
from mononn_amd import MonoNNError, MonoNNModule, binding
from mononn_amd.hlo import models
from oracle import decoding, hlo_interp


# ---- oracle -----------------------------------------------------------------------------------------------------------
def test_oracle_rope_is_a_complex_rotation():
    rng = np.random.default_rng(1)
    x, pos, f = rng.normal(size=(5, 3, 12)), np.array([0, 1, 7, 1000, 999999]), 10000.0 ** (-np.arange(4) / 4.0)
    for inter in (False, True):
        y = decoding.rope(x, pos, f, inter, 1.5)
        a, b = (x[..., 0:8:2], x[..., 1:8:2]) if inter else (x[..., :4], x[..., 4:8])
        z = (a + 1j * b) * 1.5 * np.exp(1j * pos[:, None, None] * f)
        ya, yb = (y[..., 0:8:2], y[..., 1:8:2]) if inter else (y[..., :4], y[..., 4:8])
        assert np.allclose(ya, z.real, atol=1e-9) and np.allclose(yb, z.imag, atol=1e-9)
        assert np.array_equal(y[..., 8:], x[..., 8:])


def test_oracle_attention_matches_dense_softmax():
    rng = np.random.default_rng(2)
    new, ctx, page = [3, 1, 0, 4], [9, 17, 5, 4], 4
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, page)
    kc, vc, q = rng.normal(size=(pages, page, 2, 8)), rng.normal(size=(pages, page, 2, 8)), rng.normal(size=(8, 6, 8))
    for window in (0, 3):
        got = decoding.paged_attention(q, kc, vc, table, qs, cl, 0.3, window)
        at = 0
        for b, (n, c) in enumerate(zip(new, ctx)):
            k = np.concatenate([kc[p] for p in table[b] if p >= 0])[:c]
            v = np.concatenate([vc[p] for p in table[b] if p >= 0])[:c]
            key, query = np.arange(c)[None, :], np.arange(c - n, c)[:, None]
            seen = (key <= query) & ((key > query - window) if window else True)
            for h in range(6):
                s = np.where(seen, q[at:at + n, h] @ k[:, h // 3].T * 0.3, -np.inf)
                e = np.exp(s - s.max(1, keepdims=True)) if n else s
                assert np.allclose(got[at:at + n, h], (e / e.sum(1, keepdims=True)) @ v[:, h // 3], atol=1e-12)
            at += n


def test_oracle_append_and_empty_rows():
    rng = np.random.default_rng(3)
    table, qs, cl, pages = dc.paged_batch(rng, [2, 3], [5, 2], 2)
    k, v = rng.normal(size=(6, 1, 4)), rng.normal(size=(6, 1, 4))
    kc0, vc0 = np.zeros((pages, 2, 1, 4)), np.zeros((pages, 2, 1, 4))
    kc, vc = decoding.kv_append(k, v, kc0, vc0, table, qs, cl)
    assert np.array_equal(kc[table[0, 1], 1], k[0]) and np.array_equal(kc[table[0, 2], 0], k[1])   # positions 3 and 4
    assert np.array_equal(vc[table[1, 0], 0], v[3]) and np.array_equal(vc[table[1, 0], 1], v[4])   # position -1 left out
    assert np.count_nonzero(kc.any(-1)) == 4
    o = decoding.paged_attention(rng.normal(size=(6, 2, 4)), kc, vc, table, qs, cl, 1.0)
    assert not o[2].any() and not o[5].any() and o[3].any()   # a row without keys, a token of no sequence


def test_oracle_w4_by_loops():
    rng = np.random.default_rng(4)
    x, w, s, z = rng.normal(size=(2, 64)), rng.integers(0, 256, (3, 32), dtype=np.uint8), rng.uniform(0.5, 1, (3, 2)), rng.integers(0, 16, (3, 2), dtype=np.uint8)
    for zeros in (None, z):
        got = decoding.matvec_w4(x, w, s, zeros)
        for m in range(2):
            for n in range(3):
                want = sum(x[m, k] * ((int(w[n, k // 2]) >> 4 * (k % 2) & 15) - (8 if zeros is None else int(z[n, k // 32]))) * s[n, k // 32] for k in range(64))
                assert abs(got[m, n] - want) < 1e-12


def test_hlo_oracle_runs_the_custom_calls():
    rng = np.random.default_rng(5)
    text, _ = dc.rope_module(3, 2, 8, 4, "f16", True, 0.5)
    x, pos, f = rng.normal(size=(3, 2, 8)).astype(np.float16), np.array([0, 5, 77], np.int32), np.array([1.0, 0.01], np.float32)
    assert np.array_equal(hlo_interp.evaluate(text, [x, pos, f])[0], decoding.rope(x, pos, f, True, 0.5).astype(np.float16))
    table, qs, cl, pages = dc.paged_batch(rng, [1, 2], [6, 3], 4)
    k, v = rng.normal(size=(3, 2, 16)).astype(np.float16), rng.normal(size=(3, 2, 16)).astype(np.float16)
    cache = rng.normal(size=(pages, 4, 2, 16)).astype(np.float16)
    text, _ = dc.append_module(3, 2, 16, pages, 4, 2, table.shape[1], "f16")
    kc, vc = hlo_interp.evaluate(text, [k, v, cache, cache, table, qs, cl])
    assert np.array_equal(kc, decoding.kv_append(k, v, cache, cache, table, qs, cl)[0].astype(np.float16)) and vc.dtype == np.float16
    text, _ = dc.attention_module(3, 4, 2, 16, pages, 4, 2, table.shape[1], "f16", 0.25)
    o = hlo_interp.evaluate(text, [rng.normal(size=(3, 4, 16)).astype(np.float16), kc, vc, table, qs, cl])[0]
    assert o.shape == (3, 4, 16) and np.isfinite(o.astype(np.float32)).all()


# ---- frequencies ------------------------------------------------------------------------------------------------------
def test_rope_frequencies():
    plain = models.rope_frequencies(64)
    assert plain[0] == 1.0 and plain.dtype == np.float32 and np.all(np.diff(plain) < 0)
    assert np.allclose(models.rope_frequencies(64, stretch=4.0), plain / 4.0, rtol=1e-6)
    base = models.rope_frequencies(64, stretch=4.0, method="base")
    assert base[0] == 1.0 and np.isclose(base[-1], plain[-1] / 4.0, rtol=1e-5)
    turns = models.rope_frequencies(64, stretch=4.0, method="by_turns")
    assert turns[0] == plain[0] and np.isclose(turns[-1], plain[-1] / 4.0, rtol=1e-6)
    assert np.all(turns <= plain) and np.all(turns >= plain / 4.0 * (1 - 1e-6))
    assert np.array_equal(models.rope_frequencies(64, stretch=1.0, method="by_turns"), plain)


# ---- refusals ---------------------------------------------------------------------------------------------------------
HEAD = "HloModule cluster_0__refusal.1\n\n"


def refused(body, status, words):
    with pytest.raises(MonoNNError) as err:
        MonoNNModule.compile(HEAD + "ENTRY %main {\n" + body + "\n}\n", build=False)
    assert err.value.status == status, err.value
    assert words in str(err.value), err.value


def params(*shapes):
    return "".join(f"  %p{i} = {s} parameter({i})\n" for i, s in enumerate(shapes))


def call(shape, target, n, config="{}", extra=""):
    ops = ", ".join(f"%p{i}" for i in range(n))
    return f'  {extra}%r = {shape} custom-call({ops}), custom_call_target="mononn${target}", backend_config="{config}"'


ROPE = ["f16[4,2,64]{2,1,0}", "s32[4]{0}", "f32[16]{0}"]


@pytest.mark.parametrize("shapes, result, status, words", [
    (ROPE[:2], "f16[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "takes (x, positions, inv_freq)"),
    (["f16[4,128]{1,0}"] + ROPE[1:], "f16[4,128]{1,0}", "INVALID_ARGUMENT", "[tokens, heads, head size]"),
    (["s32[4,2,64]{2,1,0}"] + ROPE[1:], "s32[4,2,64]{2,1,0}", "UNSUPPORTED", "f16, bf16 or f32"),
    ([ROPE[0], "s32[5]{0}", ROPE[2]], "f16[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "one position per token"),
    ([ROPE[0], "s64[4]{0}", ROPE[2]], "f16[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "positions must be s32"),
    ([ROPE[0], ROPE[1], "f16[16]{0}"], "f16[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "inv_freq must be f32"),
    ([ROPE[0], ROPE[1], "f32[33]{0}"], "f16[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "more pairs than a head"),
    (ROPE, "f32[4,2,64]{2,1,0}", "INVALID_ARGUMENT", "result's shape"),
    (["f16[0,2,64]{2,1,0}", "s32[0]{0}", ROPE[2]], "f16[0,2,64]{2,1,0}", "INVALID_ARGUMENT", "at least one element"),
])
def test_rope_refusals(shapes, result, status, words):
    refused(params(*shapes) + call(result, "rope", len(shapes), extra="ROOT "), status, words)


def test_config_refusals():
    refused(params(*ROPE) + call(ROPE[0], "rope", 3, '{\\"amplitude\\":1e999}', "ROOT "), "INVALID_ARGUMENT", "finite")
    att = ["f16[4,8,64]{2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "s32[3,5]{1,0}", "s32[4]{0}", "s32[3]{0}"]
    refused(params(*att) + call(att[0], "paged_attention", 6, '{\\"scale\\":1,\\"window\\":-1}', "ROOT "), "INVALID_ARGUMENT", "window")
    refused(params(*ROPE) + call(ROPE[0], "rope", 3, '{\\"amplitude\\":1e300}', "ROOT "), "INVALID_ARGUMENT", "finite")   # not in f32
    for scale in ("0", "-0.125", "1e-300"):
        refused(params(*att) + call(att[0], "paged_attention", 6, '{\\"scale\\":' + scale + '}', "ROOT "), "INVALID_ARGUMENT", "scale must be positive")


def test_a_window_of_every_key_is_no_window():
    text = [dc.attention_module(4, 8, 2, 64, 9, 16, 3, 5, "f16", 0.125, w)[0] for w in (0, 80, (1 << 31) - 1, 79)]
    src = [MonoNNModule.compile(t, build=False).get_source("main.hip") for t in text]
    assert src[0] == src[1] == src[2] != src[3]


def test_liveout_parameter_checks_its_arguments():
    m = MonoNNModule.compile(dc.append_module(5, 2, 64, 9, 3, 2, 4, "f32")[0], build=False)
    value = ctypes.c_int(7)
    ask = binding._lib.mononn_module_liveout_parameter
    assert ask(m._h, 1, ctypes.byref(value)) == 0 and value.value == 3
    for handle, index, out in ((m._h, 2, ctypes.byref(value)), (m._h, -1, ctypes.byref(value)), (m._h, 0, None), (None, 0, ctypes.byref(value))):
        assert ask(handle, index, out) == 1   # invalid argument
    assert value.value == 3


def append_and_attend(returned):
    """A module that appends to its caches (parameters 2 and 3) and attends over them; `returned` of out, kc, vc are its results."""
    def build(e):
        cache = (9, 16, 2, 64)
        a = [e.parameter("f16", (5, 2, 64), "k"), e.parameter("f16", (5, 2, 64), "v"), e.parameter("f16", cache, "k_cache"), e.parameter("f16", cache, "v_cache"),
             e.parameter("s32", (2, 4), "page_table"), e.parameter("s32", (3,), "query_start"), e.parameter("s32", (2,), "context_len")]
        kc, vc = e.kv_append(*a)
        out = e.paged_attention(e.parameter("f16", (5, 4, 64), "q"), kc, vc, *a[4:], 0.125)
        return [{"out": out, "kc": kc, "vc": vc}[r] for r in returned]
    return dc.module(build)


@pytest.mark.parametrize("returned, liveouts", [(["out"], [-1]), (["out", "vc"], [-1, 3]), (["kc", "out"], [2, -1]), (["out", "kc", "vc"], [-1, 2, 3])])
def test_updated_parameters_do_not_depend_on_what_is_returned(returned, liveouts):
    m = MonoNNModule.compile(append_and_attend(returned)[0], build=False)
    assert m.liveout_parameters() == liveouts and m.updated_parameters() == {2: "f16", 3: "f16"}


def test_parameter_updated_checks_its_arguments():
    m = MonoNNModule.compile(append_and_attend(["out"])[0], build=False)
    value, name = ctypes.c_int(7), ctypes.c_char_p()
    ask = binding._lib.mononn_module_parameter_updated
    assert ask(m._h, 3, ctypes.byref(value), None) == 0 and value.value == 1
    assert ask(m._h, 4, ctypes.byref(value), ctypes.byref(name)) == 0 and value.value == 0 and name.value == b"s32"
    value.value = 7
    for handle, index, out in ((m._h, 8, ctypes.byref(value)), (m._h, -1, ctypes.byref(value)), (m._h, 0, None), (None, 0, ctypes.byref(value))):
        assert ask(handle, index, out, None) == 1   # invalid argument
    assert value.value == 7
    assert MonoNNModule.compile(dc.rope_module(3, 5, 80, 20, "f16")[0], build=False).updated_parameters() == {}


ATT = ["f16[4,8,64]{2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "s32[3,5]{1,0}", "s32[4]{0}", "s32[3]{0}"]


@pytest.mark.parametrize("change, status, words", [
    ({0: "f16[4,7,64]{2,1,0}"}, "INVALID_ARGUMENT", "multiple of the key heads"),
    ({0: "f32[4,8,64]{2,1,0}", 1: "f32[9,16,2,64]{3,2,1,0}", 2: "f32[9,16,2,64]{3,2,1,0}"}, "UNSUPPORTED", "f16 or bf16"),
    ({1: "bf16[9,16,2,64]{3,2,1,0}"}, "INVALID_ARGUMENT", "the caches must be"),
    ({2: "f16[8,16,2,64]{3,2,1,0}"}, "INVALID_ARGUMENT", "share a shape"),
    ({0: "f16[4,8,72]{2,1,0}", 1: "f16[9,16,2,72]{3,2,1,0}", 2: "f16[9,16,2,72]{3,2,1,0}"}, "UNSUPPORTED", "multiple of 16"),
    ({0: "f16[4,8,272]{2,1,0}", 1: "f16[9,16,2,272]{3,2,1,0}", 2: "f16[9,16,2,272]{3,2,1,0}"}, "UNSUPPORTED", "multiple of 16"),
    ({3: "s64[3,5]{1,0}"}, "INVALID_ARGUMENT", "page_table"),
    ({4: "s32[3]{0}"}, "INVALID_ARGUMENT", "number of sequences"),
    ({5: "s32[4]{0}"}, "INVALID_ARGUMENT", "number of sequences"),
    ({3: "s32[3,200000000]{1,0}"}, "UNSUPPORTED", "too many"),
    ({1: "f16[9,4294967296,2,64]{3,2,1,0}", 2: "f16[9,4294967296,2,64]{3,2,1,0}", 3: "s32[3,4294967296]{1,0}"}, "UNSUPPORTED", "too many"),   # a product of 2^64
    ({1: "f16[9,33554432,2,64]{3,2,1,0}", 2: "f16[9,33554432,2,64]{3,2,1,0}", 3: "s32[3,1]{1,0}"}, "UNSUPPORTED", "a page has too many"),
])
def test_paged_attention_refusals(change, status, words):
    shapes = [change.get(i, s) for i, s in enumerate(ATT)]
    refused(params(*shapes) + call(shapes[0], "paged_attention", 6, '{\\"scale\\":1,\\"window\\":0}', "ROOT "), status, words)


APP = ["f16[4,2,64]{2,1,0}", "f16[4,2,64]{2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "f16[9,16,2,64]{3,2,1,0}", "s32[3,5]{1,0}", "s32[4]{0}", "s32[3]{0}"]
APP_RESULT = "(f16[9,16,2,64]{3,2,1,0}, f16[9,16,2,64]{3,2,1,0})"


def append_body(shapes, operands="%p0, %p1, %p2, %p3, %p4, %p5, %p6", tail=None, result=APP_RESULT, before=""):
    c = "f16[9,16,2,64]{3,2,1,0}"
    tail = tail if tail is not None else f"  %a = {c} get-tuple-element(%r), index=0\n  %b = {c} get-tuple-element(%r), index=1\n  ROOT %t = ({c}, {c}) tuple(%a, %b)"
    return params(*shapes) + before + f'  %r = {result} custom-call({operands}), custom_call_target="mononn$kv_append", backend_config="{{}}"\n' + tail


def test_kv_append_refusals():
    c = "f16[9,16,2,64]{3,2,1,0}"
    MonoNNModule.compile(HEAD + "ENTRY %main {\n" + append_body(APP) + "\n}\n", build=False)   # as it should be
    refused(append_body(APP, "%p0, %p1, %p2, %p2, %p4, %p5, %p6"), "INVALID_ARGUMENT", "different parameters")
    refused(append_body([*APP[:1], "f16[4,2,32]{2,1,0}", *APP[2:]]), "INVALID_ARGUMENT", "share a type and a shape")
    refused(append_body([*APP[:2], "f16[9,16,3,64]{3,2,1,0}", *APP[3:]]), "INVALID_ARGUMENT", "the caches must be")
    refused(append_body([*APP[:2], "f16[9,16,2,64]{2,3,1,0}", *APP[3:]]), "UNSUPPORTED", "row-major")
    refused(append_body(APP, before=f"  %copy = {c} copy(%p2)\n", operands="%p0, %p1, %copy, %p3, %p4, %p5, %p6"), "UNSUPPORTED", "entry parameters")
    # the value from before the call is also read: by another instruction, and by the call itself as its keys
    refused(append_body(APP, tail=f"  %a = {c} get-tuple-element(%r), index=0\n  %n = {c} negate(%p2)\n  ROOT %t = ({c}, {c}) tuple(%a, %n)"), "UNSUPPORTED", "updated in place")
    refused(append_body([*APP, "f32[33]{0}"], "%p0, %p1, %p2, %p3, %p4, %p5, %p6, %p7"), "INVALID_ARGUMENT", "more pairs than a head")
    refused(append_body(APP, result="(f16[9,16,2,64]{3,2,1,0}, f16[8,16,2,64]{3,2,1,0})"), "INVALID_ARGUMENT", "result's shape")


W4 = ["f16[2,256]{1,0}", "u8[48,128]{1,0}", "f16[48,2]{1,0}", "u8[48,2]{1,0}"]


@pytest.mark.parametrize("change, status, words", [
    ({0: "f32[2,256]{1,0}", 2: "f32[48,2]{1,0}"}, "UNSUPPORTED", "f16 or bf16"),
    ({1: "s8[48,128]{1,0}"}, "INVALID_ARGUMENT", "weight must be u8"),
    ({1: "u8[48,256]{1,0}"}, "INVALID_ARGUMENT", "two values to a byte"),
    ({2: "bf16[48,2]{1,0}"}, "INVALID_ARGUMENT", "scales must be"),
    ({2: "f16[48,3]{1,0}", 3: "u8[48,3]{1,0}"}, "INVALID_ARGUMENT", "scales must be"),
    ({2: "f16[48,16]{1,0}", 3: "u8[48,16]{1,0}"}, "UNSUPPORTED", "group size"),
    ({3: "u8[48,4]{1,0}"}, "INVALID_ARGUMENT", "zeros must be"),
    ({3: "f16[48,2]{1,0}"}, "INVALID_ARGUMENT", "zeros must be"),
])
def test_matvec_w4_refusals(change, status, words):
    shapes = [change.get(i, s) for i, s in enumerate(W4)]
    refused(params(*shapes) + call("f16[2,48]{1,0}", "matvec_w4", 4, extra="ROOT "), status, words)


# rows, columns, threads around the widths at which x no longer fits a workgroup's LDS: whole and in slices
W4_WIDE = [(1, 49152, 512), (1, 49280, 512), (2, 21760, 512), (2, 21888, 512), (2, 22016, 256), (2, 24576, 512), (2, 24704, 512), (3, 16384, 512), (3, 16512, 512),
           (64, 768, 512), (64, 896, 512), (64, 65536, 512), (65, 65536, 256), (64, 768, 1024), (128, 768, 1024), (128, 11008, 1024)]


@pytest.mark.parametrize("M, K, block", W4_WIDE)
def test_matvec_w4_has_a_plan_for_every_width(M, K, block):
    for dtype, group, zeros in (("f16", 32, False), ("bf16", 128, True)):
        text, _ = dc.w4_module(M, 40, K, group, dtype, zeros)
        spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
        spec["cuda_context"]["cuda_runtime_context"]["block_dim"]["x"] = block
        m = MonoNNModule.compile(text, json.dumps(spec))
        assert 0 < m.launch_dims()["smem"] <= 160 * 1024 and len(m.get_code_object()) > 0


def test_extents_beyond_32_bits_are_refused():
    big = ["f16[70000,256]{1,0}", "u8[40000,128]{1,0}", "f16[40000,2]{1,0}"]
    refused(params(*big) + call("f16[70000,40000]{1,0}", "matvec_w4", 3, extra="ROOT "), "UNSUPPORTED", "too many rows")
    wide = ["f16[1,4194304,1024]{2,1,0}", "s32[1]{0}", "f32[16]{0}"]
    refused(params(*wide) + call(wide[0], "rope", 3, extra="ROOT "), "UNSUPPORTED", "too many tokens or heads")
    c = "f16[9,1,4194304,1024]{3,2,1,0}"
    shapes = ["f16[1,4194304,1024]{2,1,0}"] * 2 + [c, c] + APP[4:6] + [APP[6]]
    refused(append_body(shapes, result=f"({c}, {c})"), "UNSUPPORTED", "too many tokens")


def test_step_counts_beyond_64_bits_are_refused():
    # 2^26 heads, 2^30 sequences (one entry of query_start more) and 8128 keys of each: 2^64 and a little in steps of 32 keys
    shapes = ["f16[1,67108864,16]{2,1,0}"] + ["f16[9,1,67108864,16]{3,2,1,0}"] * 2 + ["s32[1073741823,8128]{1,0}", "s32[1073741824]{0}", "s32[1073741823]{0}"]
    refused(params(*shapes) + call(shapes[0], "paged_attention", 6, '{\\"scale\\":1,\\"window\\":0}', "ROOT "), "UNSUPPORTED", "too many tokens times keys")


def test_other_targets_stay_refused():
    refused(params("f32[4]{0}") + call("f32[4]{0}", "paged_attention_parts", 1, extra="ROOT "), "UNSUPPORTED", "is not supported")
    refused(params("f32[4]{0}") + call("f32[4]{0}", "nothing", 1, extra="ROOT "), "UNSUPPORTED", "is not supported")


# ---- program ----------------------------------------------------------------------------------------------------------
def test_step_is_one_kernel_with_caches_in_place():
    fx = models.gpt2_step(L=2, H=128, NH=4, NKV=2, F=256, vocab=300, rotary=True, weights_4bit=32)
    m = MonoNNModule.compile(fx.hlo_text, build=False)
    assert m.liveout_parameters() == [-1, 5, 6, 7, 8]
    src = m.get_source("main.hip")
    for name in ("rope_unit", "kv_append_unit", "Attention::partial", "Attention::join", "MatvecW4"):
        # both layers share one device function each
        assert src.count("mononn_dev::" + name) + src.count(" " + name) >= 1
    assert src.count("typedef mononn_dev::PagedAttention") == 2   # its two stages
    # the cache update of a layer comes before the attention that reads it, and that before its join
    stage = {}
    for line in m.summary().splitlines():
        w = line.split()
        if w[:1] == ["stage"] and w[2] == "oper":
            stage.setdefault(w[3].split("_")[1] + ("_parts" if "parts" in w[3] else ""), []).append(int(w[1]))
    assert all(a < p < j for a, p, j in zip(stage["kv"], stage["paged_parts"], stage["paged"]))


def test_modules_without_operators_do_not_carry_them():
    m = MonoNNModule.compile(models.bert_layer(B=1, S=32, H=128, NH=4, F=256).hlo_text, build=False)
    with pytest.raises(MonoNNError):
        m.get_source("operators.h")
    assert "operators.h" not in m.get_source("main.hip")


def test_parts_have_their_own_memory():
    # two attentions in one stage and one behind them; and the result is written from the stage of the parts on
    def build(e):
        cache, meta = ("f16", (20, 16, 2, 64)), [("s32", (2, 8)), ("s32", (3,)), ("s32", (2,))]
        caches = [e.parameter(*cache, f"c{i}") for i in range(4)]
        t, s, c = [e.parameter(*m, "m") for m in meta]
        q = e.parameter("f16", (2, 4, 64), "q")
        a, b = e.paged_attention(q, caches[0], caches[1], t, s, c, 0.1), e.paged_attention(q, caches[2], caches[3], t, s, c, 0.1)
        return e.paged_attention(e.binary("add", a, b), caches[0], caches[3], t, s, c, 0.1)
    text, _ = dc.module(build)
    for barrier in ("flags_coherent", "flags"):
        spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
        spec["mononn_hip"]["barrier"] = barrier
        m = MonoNNModule.compile(text, json.dumps(spec), build=False)
        part = 2 * 256 * (16 * 64 + 32) * 4   # two parts per workgroup, 16 rows of 64 elements each with a maximum and a sum
        assert m.buffer_info()["temp"] >= 2 * part


def between_units(source):
    """The statements of the kernel's unit loop in front of its dispatch, and the calls that have LDS to wait for."""
    kernel = source[source.index('extern "C"'):]
    loop = kernel[kernel.index("const int unit = u - first;"):]
    return loop[:loop.index("switch (fn)")], [line for line in kernel.splitlines() if "lds_shared = true" in line]


def test_units_of_a_stage_do_not_meet_in_the_lds():
    # 224 units of a 4-bit product and 64 of a LayerNorm on 256 workgroups: 32 of them go from the one, whose waves end with
    # reads of the LDS, to the other, which begins with stores there
    def build(e):
        y = e.matvec_w4(e.parameter("f16", (1, 128), "x"), e.parameter("u8", (14336, 64), "w"), e.parameter("f16", (14336, 1), "s"))
        h, g, b = e.parameter("f16", (64, 768), "h"), e.parameter("f16", (768,), "g"), e.parameter("f16", (768,), "b")
        return y, models._layer_norm(e, e.module, h, g, b, 1e-5)
    m = MonoNNModule.compile(dc.module(build)[0], build=False)
    assert "stages=1 nodes=2" in m.summary()
    loop, calls = between_units(m.get_source("main.hip"))
    assert "if (lds_shared && worked) __syncthreads();" in loop and "worked = true;" in loop
    assert len(calls) == 1 and "units = 64; first = 224; total = 288;" in calls[0]


def test_a_gemm_behind_its_row_program_waits_for_its_own_last_unit():
    # k split over waves: a unit ends with reads of the sums in the LDS, the next one begins with the row program's exchange there
    def build(e):
        h, g, b = e.parameter("f16", (1024, 256), "h"), e.parameter("f16", (256,), "g"), e.parameter("f16", (256,), "b")
        return e.gemm(models._layer_norm(e, e.module, h, g, b, 1e-5), e.parameter("f16", (256, 1024), "w"), 1, 0)
    text = dc.module(build)[0]
    spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
    spec["mononn_hip"]["gemm_prologue_fusion"] = True
    for nodes in ("gemm_spec_list", "cluster_reduce_spec", "cluster_elewise_spec"):
        spec[nodes] = {}
    spec = json.loads(MonoNNModule.compile(text, json.dumps(spec), build=False).get_tuning_spec())
    (gemm,) = spec["gemm_spec_list"].values()
    for waves_k, wait in ((4, True), (1, False)):
        gemm["cutlass_config"].update(threadblockshape={"m": 32, "n": 32, "k": 32}, warpshape={"m": 32 if waves_k == 4 else 16, "n": 32 if waves_k == 4 else 16, "k": 256 // waves_k},
                                      wave_arrangement={"m": 1 if waves_k == 4 else 2, "n": 1 if waves_k == 4 else 2, "k": waves_k})
        m = MonoNNModule.compile(text, json.dumps(spec))
        assert "+row-prologue" in m.summary() and m.launch_dims()["grid"] == 256
        loop, calls = between_units(m.get_source("main.hip"))
        assert len(calls) == (1 if wait else 0) and ("__syncthreads" in loop) == wait


@pytest.mark.parametrize("T, H, HKV, D, block", [(5, 32, 8, 128, None), (32, 32, 8, 128, None), (4000, 32, 8, 128, None), (4, 8, 1, 256, None), (90, 4, 4, 64, 1024)])
def test_parts_of_attention_fit_the_static_arena(T, H, HKV, D, block):
    text = dc.attention_module(T, H, HKV, D, 90, 16, 4, 300, "bf16", 0.1)[0]
    spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
    if block:
        spec["cuda_context"]["cuda_runtime_context"]["block_dim"]["x"] = block
    m = MonoNNModule.compile(text, json.dumps(spec), build=False)
    waves, rows = (block or 512) // 64, T * H // HKV
    part = min(waves, -(-rows // 32)) * (D // 32 * 1024 + 64) * 4   # per block of 32 rows: its output, maxima and sums
    assert 2 * 256 * part <= m.buffer_info()["temp"] <= binding._lib.mononn_static_temp_bytes()
    assert m.buffer_info()["temp"] < 2 * 256 * part + 4096


# ---- every variant builds -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("text", [
    dc.rope_module(3, 5, 80, 20, "bf16", True)[0], dc.rope_module(7, 3, 10, 6, "f32")[0], dc.append_module(5, 2, 64, 9, 3, 2, 4, "f32")[0],
    dc.attention_module(70, 8, 2, 80, 90, 8, 3, 20, "bf16", 0.1, 100)[0], dc.attention_module(40, 4, 4, 256, 90, 8, 2, 20, "f16", 0.1)[0],
    dc.attention_module(2, 2, 1, 16, 9, 1, 2, 20, "f16", 0.1)[0], dc.w4_module(70, 33, 640, 32, "bf16", True)[0], dc.w4_module(1, 100, 96, 32, "f16", False)[0]])
def test_builds_for_the_gpu(text):
    for block in (64, 256, 512):
        spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
        spec["cuda_context"]["cuda_runtime_context"]["block_dim"]["x"] = block
        assert len(MonoNNModule.compile(text, json.dumps(spec)).get_code_object()) > 0


# ---- bounds -----------------------------------------------------------------------------------------------------------
HERE = os.path.dirname(os.path.abspath(__file__))
FILL = "for (size_t k = 0; k < sizes[i]; ++k) base[k] = char(k * 7 + i);     // finite halves, small integers as indices"


def check(monkeypatch, tmp_path, text, data=None, grid=None, block=None, shrink=None):
    """cpu_bounds.check_module with the operators' header and host builtins; data: parameter number -> s32 contents."""
    m = MonoNNModule.compile(text, build=False)
    spec = json.loads(m.get_tuning_spec())
    launch = spec["cuda_context"]["cuda_runtime_context"]
    launch["grid_dim"]["x"], launch["block_dim"]["x"] = grid or launch["grid_dim"]["x"], block or launch["block_dim"]["x"]
    (tmp_path / "operators.h").write_text(m.get_source("operators.h"))
    for i, a in (data or {}).items():
        np.asarray(a, np.int32).tofile(str(tmp_path / f"param_{i}.bin"))
    assert FILL in cpu_bounds.DRIVER
    read = FILL + ('\n    if (FILE* f = std::fopen((std::string("' + str(tmp_path) + '/param_") + std::to_string(i) + ".bin").c_str(), "rb")) '
                   "{ const size_t n = std::fread(base, 1, sizes[i], f); (void)n; std::fclose(f); }")
    monkeypatch.setattr(cpu_bounds, "DRIVER", cpu_bounds.DRIVER.replace(FILL, read).replace("#include <csignal>", "#include <csignal>\n#include <string>"))
    monkeypatch.setattr(cpu_bounds, "HERE", os.path.join(HERE, "cpu_shim", "operators"))
    return cpu_bounds.check_module(text, json.dumps(spec), workdir=str(tmp_path), opt="-O1", shrink=shrink)


def any_pages(rng, B, W, pages):
    return rng.integers(-3, pages + 3, (B, W))


@pytest.mark.parametrize("T, H, D, R, dtype, inter", [(3, 5, 80, 20, "f16", False), (33, 12, 64, 16, "f32", True), (1, 1, 2, 2, "bf16", False), (9, 3, 10, 6, "f32", False), (700, 32, 128, 128, "bf16", True)])
def test_bounds_rope(monkeypatch, tmp_path, T, H, D, R, dtype, inter):
    assert check(monkeypatch, tmp_path, dc.rope_module(T, H, D, R, dtype, inter)[0]) == (True, "ok")


@pytest.mark.parametrize("qs, cl", [([0, 5, 30, 37], [32, 25, 7]), ([0, 5, 30, 37], [40, 25, 7]), ([2, 1, -9, 99], [40, -3, 1 << 30]), ([0, 0, 0, 0], [1, 2, 3]), ([0, 37, 37, 37], [30, 0, 0])])
@pytest.mark.parametrize("R", [0, 40])
def test_bounds_append(monkeypatch, tmp_path, qs, cl, R):
    rng = np.random.default_rng(6)
    assert check(monkeypatch, tmp_path, dc.append_module(37, 3, 80, 9, 8, 3, 4, "bf16", R)[0], {4: any_pages(rng, 3, 4, 9), 5: qs, 6: cl}) == (True, "ok")


@pytest.mark.parametrize("T, H, HKV, D, B, W, page, window, block, qs, cl", [
    (4, 12, 12, 64, 4, 8, 16, 0, 256, [0, 1, 2, 3, 4], [1, 128, 77, 0]),
    (70, 8, 2, 80, 3, 20, 8, 100, 512, [0, 3, 60, 69], [160, 99, 12]),
    (70, 8, 2, 80, 3, 20, 8, 0, 256, [2, 3, 60, 1000], [170, 3, 12]),
    (40, 4, 4, 256, 2, 20, 8, 0, 256, [0, 39, 40], [170, 30]),
    (9, 4, 2, 256, 2, 20, 8, 7, 512, [0, 8, 9], [170, 30]),
    (5, 3, 1, 16, 2, 9, 1, 0, 64, [0, 5, 3], [-4, 1 << 30]),
    (130, 2, 2, 96, 1, 30, 5, 0, 128, [0, 130], [149]),
    (600, 8, 2, 64, 3, 90, 8, 33, 1024, [0, 1, 520, 600], [160, 719, 80]),
])
def test_bounds_attention(monkeypatch, tmp_path, T, H, HKV, D, B, W, page, window, block, qs, cl):
    rng = np.random.default_rng(7)
    text, _ = dc.attention_module(T, H, HKV, D, 30, page, B, W, "bf16", 0.1, window)
    assert check(monkeypatch, tmp_path, text, {3: any_pages(rng, B, W, 30), 4: qs, 5: cl}, grid=8, block=block) == (True, "ok")


@pytest.mark.parametrize("T, H, HKV, D, B, W, page, window, block, qs, cl, whole", [
    (4, 4, 2, 64, 4, 8, 16, 0, 256, [0, 1, 2, 3, 4], [1, 128, 77, 0], True),          # single tokens
    (4, 4, 2, 64, 4, 32, 16, 0, 256, [0, 1, 2, 3, 4], [1, 500, 77, 0], False),        # one of them long
    (70, 8, 2, 80, 3, 20, 8, 0, 256, [0, 70, 70, 70], [70, 99, 12], True),            # one prompt
    (70, 8, 2, 80, 3, 20, 8, 30, 512, [0, 3, 3, 70], [100, 99, 90], True),            # a few tokens and a prompt, with a window
    (70, 8, 2, 80, 3, 20, 8, 0, 256, [2, 3, 60, 1000], [1 << 30, -3, 12], True),      # lengths that are cut to the table and the tokens
    (70, 8, 2, 80, 3, 90, 8, 0, 256, [0, 3, 60, 70], [700, 99, 12], False),           # a cache that one range would work on for long
    (40, 4, 4, 256, 2, 20, 8, 0, 256, [0, 39, 40], [60, 30], True),
])
def test_bounds_attention_of_uncut_items(monkeypatch, tmp_path, T, H, HKV, D, B, W, page, window, block, qs, cl, whole):
    # items that are not cut leave no parts: without memory for them the run still ends well, and only then
    rng = np.random.default_rng(8)
    text, _ = dc.attention_module(T, H, HKV, D, 30, page, B, W, "f16", 0.1, window)
    spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
    launch = spec["cuda_context"]["cuda_runtime_context"]
    launch["grid_dim"]["x"], launch["block_dim"]["x"] = 8, block
    parts = MonoNNModule.compile(text, json.dumps(spec), build=False).buffer_info()["temp"]
    data = {3: any_pages(rng, B, W, 30), 4: qs, 5: cl}
    ok, message = check(monkeypatch, tmp_path, text, data, grid=8, block=block, shrink=("temp arena", parts))
    assert ok == whole and (ok or "temp arena" in message), message


@pytest.mark.parametrize("M, N, K, group, dtype, zeros", [(1, 100, 96, 32, "f16", False), (19, 33, 640, 32, "bf16", True), (70, 33, 256, 128, "f16", True), (3, 16, 64, 64, "bf16", False), (1, 1, 1280, 256, "f16", True),
                                                         (16, 40, 4096, 64, "f16", True), (70, 33, 1056, 32, "bf16", False)])   # x in slices
def test_bounds_w4(monkeypatch, tmp_path, M, N, K, group, dtype, zeros):
    assert check(monkeypatch, tmp_path, dc.w4_module(M, N, K, group, dtype, zeros)[0], grid=8) == (True, "ok")


@pytest.mark.parametrize("M, K, group, block", [(2, 21888, 32, 256), (64, 768, 32, 1024), (65, 65536, 128, 256)])
def test_bounds_w4_of_wide_x(monkeypatch, tmp_path, M, K, group, block):
    assert check(monkeypatch, tmp_path, dc.w4_module(M, 20, K, group, "f16", True)[0], grid=8, block=block) == (True, "ok")


def test_bounds_harness_sees_the_operators(monkeypatch, tmp_path):
    text, _ = dc.append_module(5, 2, 64, 9, 3, 2, 4, "f32")
    ok, message = check(monkeypatch, tmp_path, text, {4: [[8] * 4, [0] * 4], 5: [0, 1, 5], 6: [6, 4]}, shrink=("parameter 2", 16))
    assert not ok and "parameter 2" in message
    text, _ = dc.attention_module(4, 12, 12, 64, 30, 16, 4, 8, "f16", 0.1)
    ok, message = check(monkeypatch, tmp_path, text, {3: [[29] * 8] * 4, 4: [0, 1, 2, 3, 4], 5: [1, 128, 77, 0]}, grid=8, block=256, shrink=("LDS", 4096))
    assert not ok and "LDS" in message
