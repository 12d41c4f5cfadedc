"""The decoding operators on the GPU against their definitions in 64 bits, element by element within bounds derived from
the roundings they make (tests/decoding_cases.py), at the sizes where tiles, pages and sequences end."""
import json

import numpy as np
import pytest

import decoding_cases as dc
from mononn_amd import MonoNNModule
from mononn_amd.hlo import models
from oracle import decoding, hlo_interp

pytestmark = pytest.mark.gpu


def run(text, outputs, inputs, block=None, grid=None):
    spec = None
    if block:
        spec = json.loads(MonoNNModule.compile(text, build=False).get_tuning_spec())
        launch = spec["cuda_context"]["cuda_runtime_context"]
        launch["block_dim"]["x"], launch["grid_dim"]["x"] = block, grid or launch["grid_dim"]["x"]
        spec = json.dumps(spec)
    m = MonoNNModule.compile(text, spec)
    m.load(0)
    out = m.run(inputs, outputs)
    m.close()
    return out


def within(got, want, bound):
    err = np.abs(got - want)
    assert np.all(np.isfinite(got)), "not finite"
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert np.all(err <= bound), f"off by {err[worst]} at {worst} where {bound[worst]} is allowed (value {want[worst]})"


# ---- rope -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T, H, D, R, dtype, inter, far", [
    (1, 32, 128, 128, "f16", False, 100000), (1, 1, 2, 2, "f32", True, 10), (997, 12, 64, 16, "f32", True, 1000000), (130, 3, 80, 20, "bf16", False, 1000000),
    (33, 5, 96, 96, "f16", True, 4096), (7, 3, 10, 6, "f32", False, 100), (2500, 32, 128, 64, "bf16", False, 1 << 30), (5, 1, 1024, 1024, "f16", False, 100), (64, 7, 72, 36, "f16", False, 5000)])
def test_rope(gpu_device, T, H, D, R, dtype, inter, far):
    rng = np.random.default_rng(11)
    text, outs = dc.rope_module(T, H, D, R, dtype, inter, 1.25)
    x, pos, f = dc.bits(rng.normal(size=(T, H, D)), dtype), rng.integers(0, far, T).astype(np.int32), models.rope_frequencies(R)
    pos[0] = 0
    (got,) = run(text, outs, [x, pos, f])
    xv = dc.values(x, dtype)
    want = decoding.rope(xv, pos, f, inter, 1.25)
    within(dc.values(got, dtype), want, dc.rotation_bound(xv, R, dtype, inter, 1.25, want))
    assert np.array_equal(got[..., R:], x[..., R:])
    # position 0 turns by nothing, with amplitude 1 bit for bit
    text, outs = dc.rope_module(T, H, D, R, dtype, inter)
    (same,) = run(text, outs, [x, np.zeros(T, np.int32), f])
    assert np.array_equal(same, x)


def test_rope_negative_positions_turn_back(gpu_device):
    rng = np.random.default_rng(12)
    text, outs = dc.rope_module(50, 2, 64, 64, "f32")
    x, pos, f = rng.normal(size=(50, 2, 64)).astype(np.float32), rng.integers(0, 10000, 50).astype(np.int32), models.rope_frequencies(64)
    (there,) = run(text, outs, [x, pos, f])
    (back,) = run(text, outs, [there, -pos, f])
    assert np.abs(back - x).max() < 1e-5


@pytest.mark.parametrize("amplitude", [1.0, 1.2079441541679836])
def test_rotation_next_to_half_a_turn(gpu_device, amplitude):
    # sines of angles within 0.01 of pi: their 32-bit angle is off by up to 9e-8, their value by four units of its last place
    # at most when what that leaves is taken into account (two of the function, one each of the further turn and the rounding).
    # The reduction itself is in 64 bits: 1 / pi and its product with the angle are rounded by 2^-53 each, which is 2^-52 of
    # the angle before its whole turns are taken off (1.7e-10 of 7.4e5 rad).
    f = np.array([0.7071, 0.0123], np.float32)
    turns = np.arange(1, 1 << 20)[:, None] * f.astype(np.float64) / (2 * np.pi) % 1.0
    pos = np.concatenate([np.nonzero(np.abs(turns[:, i] - 0.5) < 1.5e-3)[0][-200:] + 1 for i in range(2)]).astype(np.int32)
    near = np.abs(turns[pos - 1] - 0.5) < 1.5e-3
    assert near.sum(0).min() >= 200
    text, outs = dc.rope_module(len(pos), 1, 4, 4, "f32", False, amplitude)
    x = np.zeros((len(pos), 1, 4), np.float32)
    x[..., :2] = 1.0
    (got,) = run(text, outs, [x, pos, f])
    want = decoding.rope(x, pos, f, False, amplitude)
    sines, exact = got[:, 0, 2:].astype(np.float64)[near], want[:, 0, 2:][near]
    angle = (pos.astype(np.float64)[:, None] * f)[near]
    within(sines, exact, 4 * 2.0 ** -23 * np.abs(exact) + amplitude * 2.0 ** -52 * angle + 1e-13)


# ---- append -----------------------------------------------------------------------------------------------------------
APPEND = [
    dict(new=[1] * 5, ctx=[1, 2, 16, 17, 300], H=8, D=128, page=16, R=128, dtype="f16"),
    dict(new=[37, 0, 1, 64], ctx=[37, 9, 1, 100], H=3, D=80, page=8, R=40, dtype="bf16"),
    dict(new=[5, 2], ctx=[3, 2], H=2, D=64, page=3, R=0, dtype="f32"),                       # more new tokens than keys: the first two left out
    dict(new=[300, 511], ctx=[1000, 511], H=12, D=64, page=64, R=16, dtype="f32", inter=True),
    dict(new=[1], ctx=[1], H=1, D=2, page=1, R=2, dtype="f16"),
    dict(new=[3, 4], ctx=[10, 12], H=5, D=10, page=4, R=6, dtype="bf16", tokens=12),         # tokens of no sequence
]


@pytest.mark.parametrize("c", APPEND)
def test_kv_append(gpu_device, c):
    rng = np.random.default_rng(13)
    table, qs, cl, pages = dc.paged_batch(rng, c["new"], c["ctx"], c["page"])
    T, H, D, dt, R, inter = c.get("tokens", sum(c["new"])), c["H"], c["D"], c["dtype"], c["R"], c.get("inter", False)
    text, outs = dc.append_module(T, H, D, pages, c["page"], len(c["new"]), table.shape[1], dt, R, inter, 0.75)
    k, v = dc.bits(rng.normal(size=(T, H, D)), dt), dc.bits(rng.normal(size=(T, H, D)), dt)
    kc, vc = dc.bits(rng.normal(size=(pages, c["page"], H, D)), dt), dc.bits(rng.normal(size=(pages, c["page"], H, D)), dt)
    f = models.rope_frequencies(R) if R else None
    got_k, got_v = run(text, outs, [k, v, kc, vc, table, qs, cl] + ([f] if R else []))
    kv = dc.values(k, dt)
    # the same append of bit patterns: values exactly, untouched rows exactly
    want_k, want_v = decoding.kv_append(kv, dc.values(v, dt), dc.values(kc, dt), dc.values(vc, dt), table, qs, cl, f, inter, 0.75)
    assert np.array_equal(dc.values(got_v, dt), want_v)
    written = np.zeros((pages, c["page"]), bool)
    bound = np.zeros((pages, c["page"], H, D))
    for b, (start, n, ctx) in enumerate(decoding.sequences(qs, cl, T, table.shape[1] * c["page"])):
        for i in range(n):
            p = ctx - n + i
            if p >= 0:
                at = table[b, p // c["page"]], p % c["page"]
                written[at] = True
                if R:
                    row = kv[start + i][None]
                    bound[at] = dc.rotation_bound(row, R, dt, inter, 0.75, want_k[at][None])[0]
    assert written.sum() == sum(min(n, x) for n, x in zip(c["new"], c["ctx"]))
    assert np.array_equal(got_k[~written], kc[~written]) and np.array_equal(got_v[~written], vc[~written])
    within(dc.values(got_k, dt), want_k, bound)


def test_kv_append_leaves_out_bad_pages(gpu_device):
    rng = np.random.default_rng(14)
    table = np.array([[0, -1, 7], [2, 100000, -5], [-(1 << 31), (1 << 31) - 1, 3]], np.int32)
    qs, cl = np.array([0, 6, 12, 18], np.int32), np.array([6, 5, 60], np.int32)   # the last length is cut to the table's 6 positions
    text, outs = dc.append_module(18, 1, 16, 5, 2, 3, 3, "f16")
    k, v = rng.normal(size=(18, 1, 16)).astype(np.float16), rng.normal(size=(18, 1, 16)).astype(np.float16)
    kc, vc = np.zeros((5, 2, 1, 16), np.float16), np.zeros((5, 2, 1, 16), np.float16)
    got_k, got_v = run(text, outs, [k, v, kc, vc, table, qs, cl])
    want_k, want_v = decoding.kv_append(k, v, kc, vc, table, qs, cl)
    assert np.array_equal(got_k, want_k.astype(np.float16)) and np.array_equal(got_v, want_v.astype(np.float16))
    # positions 0, 1 of the first (page 0), 0, 1 of the second (page 2; its first token has position -1), 4, 5 of the third (page 3)
    assert np.count_nonzero(got_k.any((-1, -2))) == 2 + 2 + 2


# ---- attention --------------------------------------------------------------------------------------------------------
ATTENTION = [
    dict(new=[1, 1, 1, 1], ctx=[1, 33, 128, 511], H=12, HKV=12, D=64, page=16, dtype="f16"),
    dict(new=[1], ctx=[1], H=1, HKV=1, D=16, page=1, dtype="bf16"),
    dict(new=[1] * 7, ctx=[5, 700, 64, 31, 32, 2000, 1], H=32, HKV=8, D=128, page=16, dtype="bf16"),
    dict(new=[1], ctx=[9001], H=8, HKV=1, D=128, page=32, dtype="f16"),
    dict(new=[1, 1], ctx=[777, 130], H=14, HKV=2, D=80, page=8, dtype="f16"),
    dict(new=[1, 1, 1], ctx=[600, 100, 99], H=32, HKV=2, D=96, page=64, dtype="bf16", window=100),
    dict(new=[130], ctx=[130], H=4, HKV=4, D=64, page=16, dtype="f16"),
    dict(new=[65, 1, 0, 300, 17], ctx=[65, 900, 12, 1203, 17], H=8, HKV=2, D=128, page=16, dtype="bf16"),
    dict(new=[257, 64], ctx=[300, 64], H=6, HKV=2, D=80, page=7, dtype="f16", window=50),
    dict(new=[33, 2], ctx=[100, 3], H=3, HKV=3, D=256, page=16, dtype="bf16"),
    dict(new=[16, 1, 5], ctx=[300, 400, 5], H=2, HKV=1, D=256, page=16, dtype="f16"),
    dict(new=[40, 3, 9], ctx=[10, 3, 0], H=4, HKV=2, D=32, page=4, dtype="f16"),                  # rows that see no key
    dict(new=[5, 70, 1], ctx=[50, 90, 20], H=4, HKV=2, D=48, page=16, dtype="bf16", tokens=90),     # tokens of no sequence
    dict(new=[1] * 150, ctx=[1 + 7 * i % 300 for i in range(150)], H=4, HKV=2, D=64, page=16, dtype="f16"),   # more sequences than lanes
    dict(new=[20, 20], ctx=[1500, 40], H=20, HKV=1, D=112, page=16, dtype="f16", window=1),
]


@pytest.mark.parametrize("block", [256, 512])
@pytest.mark.parametrize("c", ATTENTION)
def test_paged_attention(gpu_device, c, block):
    rng = np.random.default_rng(15)
    table, qs, cl, pages = dc.paged_batch(rng, c["new"], c["ctx"], c["page"])
    T, H, HKV, D, dt, window = c.get("tokens", sum(c["new"])), c["H"], c["HKV"], c["D"], c["dtype"], c.get("window", 0)
    scale = 1.0 / np.sqrt(D)
    text, outs = dc.attention_module(T, H, HKV, D, pages, c["page"], len(c["new"]), table.shape[1], dt, scale, window)
    q = dc.bits(rng.normal(size=(T, H, D)) * 2, dt)
    kc, vc = dc.bits(rng.normal(size=(pages, c["page"], HKV, D)), dt), dc.bits(rng.normal(size=(pages, c["page"], HKV, D)), dt)
    mags = {}
    want = decoding.paged_attention(dc.values(q, dt), dc.values(kc, dt), dc.values(vc, dt), table, qs, cl, scale, window, mags)
    # cells that hold no key of a sequence are not a number
    used = np.zeros((pages, c["page"]), bool)
    for b, x in enumerate(c["ctx"]):
        for p in range(x):
            used[table[b, p // c["page"]], p % c["page"]] = True
    nan = dc.bits(np.full((1,), np.nan), dt)[0]
    kc[~used], vc[~used] = nan, nan
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl], block)
    within(dc.values(got, dt), want, dc.attention_bound(want, mags, D, dt))
    empty = ~mags["weighted"].any(-1)
    assert not dc.values(got, dt)[empty].any()


@pytest.mark.parametrize("block, grid", [(64, 256), (128, 100), (512, 128), (1024, 256), (256, 1)])
def test_paged_attention_of_other_launches(gpu_device, block, grid):
    # few and many ranges, waves and keys per step
    rng = np.random.default_rng(36)
    new, ctx, page, H, HKV, D = [65, 1, 0, 300, 17], [65, 900, 12, 1203, 17], 16, 8, 2, 128
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, page)
    for T in (sum(new), 5):
        starts = qs if T > 5 else np.arange(6, dtype=np.int32)
        lens = cl if T > 5 else np.minimum(cl, 1000)
        text, outs = dc.attention_module(T, H if T > 5 else 4, HKV, D, pages, page, 5, table.shape[1], "bf16", 0.09)
        q, kc, vc = (dc.bits(rng.normal(size=s), "bf16") for s in ((T, H if T > 5 else 4, D), (pages, page, HKV, D), (pages, page, HKV, D)))
        mags = {}
        want = decoding.paged_attention(dc.values(q, "bf16"), dc.values(kc, "bf16"), dc.values(vc, "bf16"), table, starts, lens, 0.09, 0, mags)
        (got,) = run(text, outs, [q, kc, vc, table, starts, lens], block, grid)
        within(dc.values(got, "bf16"), want, dc.attention_bound(want, mags, D, "bf16"))


def test_paged_attention_large_scores_and_one_sided_weights(gpu_device):
    # one key outweighs all others, at the first, a middle and the last position; scores of several thousand
    rng = np.random.default_rng(16)
    D, page, ctx = 64, 16, 1000
    table, qs, cl, pages = dc.paged_batch(rng, [1, 1, 40], [ctx] * 3, page)
    text, outs = dc.attention_module(42, 2, 1, D, pages, page, 3, table.shape[1], "f16", 1.0)
    q = np.full((42, 2, D), 4.0, np.float16)
    kc = np.full((pages, page, 1, D), -8.0, np.float16)
    vc = rng.normal(size=(pages, page, 1, D)).astype(np.float16)
    peaks = [0, 500, 960]
    for b, p in enumerate(peaks):
        kc[table[b, p // page], p % page] = 8.0
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl])
    for t in range(42):
        b = min(t, 2)
        assert np.array_equal(got[t, 0], vc[table[b, peaks[b] // page], peaks[b] % page, 0])


def test_paged_attention_of_bad_pages_reads_inside_the_pool(gpu_device):
    rng = np.random.default_rng(17)
    table = np.array([[0, -1, 100, 2], [(1 << 31) - 1, -(1 << 31), 1, 3]], np.int32)
    qs, cl = np.array([0, 1, 50], np.int32), np.array([16, 1 << 30], np.int32)
    text, outs = dc.attention_module(50, 2, 1, 32, 4, 4, 2, 4, "f16", 0.2)
    q, kc, vc = (rng.normal(size=s).astype(np.float16) for s in ((50, 2, 32), (4, 4, 1, 32), (4, 4, 1, 32)))
    mags = {}
    want = decoding.paged_attention(q, kc, vc, table, qs, cl, 0.2, 0, mags)
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl])
    within(got.astype(np.float64), want, dc.attention_bound(want, mags, 32, "f16"))


def test_paged_attention_page_addresses_beyond_32_bits(gpu_device):
    """A pool of 5 GiB per cache: the pages that are used lie at its end, behind 2^31 and 2^32 bytes and 2^31 elements."""
    import torch
    from mononn_amd.torch_op import MonoNNFunction
    page, HKV, D, pages, T, H, ctx = 64, 8, 128, 40960, 2, 16, 150
    assert pages * page * HKV * D > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(18)
    kc = torch.zeros((pages, page, HKV, D), dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    used = [pages - 1, pages - 2, 0, 16384, 32768, pages - 3]
    for p in used:
        kc[p].normal_(generator=g)
        vc[p].normal_(generator=g)
    table = np.array([used[:3], used[3:]], np.int32)
    qs, cl = np.array([0, 1, 2], np.int32), np.array([ctx, ctx + 1], np.int32)
    q = torch.randn((T, H, D), generator=g, device="cuda").half()
    small_k, small_v = kc[used].cpu().numpy(), vc[used].cpu().numpy()
    local = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    dev = lambda a: torch.from_numpy(a).cuda()
    text, outs = dc.attention_module(T, H, HKV, D, pages, page, 2, 3, "f16", 0.09)
    m = MonoNNModule.compile(text)
    m.load(0)
    (got,) = MonoNNFunction(m, outs, checked=True)(q, kc, vc, dev(table), dev(qs), dev(cl))
    mags = {}
    want = decoding.paged_attention(q.cpu().numpy(), small_k, small_v, local, qs, cl, 0.09, 0, mags)
    within(got.cpu().numpy().astype(np.float64), want, dc.attention_bound(want, mags, D, "f16"))
    # and an append there
    k, v = torch.randn((T, HKV, D), generator=g, device="cuda").half(), torch.randn((T, HKV, D), generator=g, device="cuda").half()
    text, outs = dc.append_module(T, HKV, D, pages, page, 2, 3, "f16")
    a = MonoNNModule.compile(text)
    a.load(0)
    ck, cv = MonoNNFunction(a, outs, checked=True)(k, v, kc, vc, dev(table), dev(qs), dev(cl))
    assert ck.data_ptr() == kc.data_ptr() and cv.data_ptr() == vc.data_ptr()
    want_k, want_v = decoding.kv_append(k.cpu().numpy(), v.cpu().numpy(), small_k, small_v, local, qs, cl)
    assert np.array_equal(kc[used].cpu().numpy(), want_k.astype(np.float16)) and np.array_equal(vc[used].cpu().numpy(), want_v.astype(np.float16))
    assert torch.count_nonzero(kc).item() == np.count_nonzero(want_k)
    a.close()
    m.close()


@pytest.mark.parametrize("block", [256, 512])
def test_paged_attention_cells_before_the_window_may_hold_anything(gpu_device, block):
    # pages that a sliding window has left are given back: not in the table any more, or written by others
    rng = np.random.default_rng(34)
    new, ctx, page, window, H, HKV, D = [1, 9, 70, 1, 200], [500, 300, 400, 64, 333], 16, 37, 4, 2, 64
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, page)
    text, outs = dc.attention_module(sum(new), H, HKV, D, pages, page, len(new), table.shape[1], "f16", 0.125, window)
    q, kc, vc = (rng.normal(size=s).astype(np.float16) for s in ((sum(new), H, D), (pages, page, HKV, D), (pages, page, HKV, D)))
    mags = {}
    want = decoding.paged_attention(q, kc, vc, table, qs, cl, 0.125, window, mags)
    seen = np.zeros((pages, page), bool)
    for b, (n, x) in enumerate(zip(new, ctx)):
        first = max(0, x - n - window + 1)
        for p in range(first, x):
            seen[table[b, p // page], p % page] = True
        table[b, :first // page] = rng.choice([-1, 0, pages + 5], first // page)
    kc[~seen], vc[~seen] = np.nan, np.inf
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl], block)
    within(got.astype(np.float64), want, dc.attention_bound(want, mags, D, "f16"))


def test_paged_attention_without_new_tokens(gpu_device):
    rng = np.random.default_rng(35)
    for H in (4, 40):   # at most 16 rows in all, and more
        text, outs = dc.attention_module(3, H, 2, 64, 9, 16, 2, 4, "f16", 0.125)
        a = [rng.normal(size=s).astype(np.float16) for s in ((3, H, 64), (9, 16, 2, 64), (9, 16, 2, 64))]
        (got,) = run(text, outs, a + [np.zeros((2, 4), np.int32), np.zeros(3, np.int32), np.array([50, 3], np.int32)])
        assert not got.any()


@pytest.mark.parametrize("block", [256, 512])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 30])
def test_paged_attention_of_values_that_cancel(gpu_device, n, dtype, block):
    # few keys of opposite values: what is left of them shows every bit that a weight has lost on the way
    rng = np.random.default_rng(46)
    H, D, page, B = 2, 16, 8, 24
    new, ctx = [n] * B, [n + 1 + 2 * i for i in range(B)]
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, page)
    text, outs = dc.attention_module(sum(new), H, H, D, pages, page, B, table.shape[1], dtype, 0.25)
    q, kc = dc.bits(rng.normal(size=(sum(new), H, D)), dtype), dc.bits(rng.normal(size=(pages, page, H, D)), dtype)
    vc = dc.bits(rng.choice([-1.0, 1.0], (pages, page, H, D)), dtype)
    mags = {}
    want = decoding.paged_attention(dc.values(q, dtype), dc.values(kc, dtype), dc.values(vc, dtype), table, qs, cl, 0.25, 0, mags)
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl], block)
    within(dc.values(got, dtype), want, dc.split_attention_bound(want, mags, D, dtype))


@pytest.mark.parametrize("n", [1, 20])
def test_paged_attention_counts_keys_far_below_the_maximum(gpu_device, n):
    # f16: one key that outweighs each of the others by 2^26, which together are a five-hundredth of it; one workgroup, whose
    # waves see all of them
    D, page, ctx = 16, 32, 131072
    rng = np.random.default_rng(47)
    table, qs, cl, pages = dc.paged_batch(rng, [n], [ctx], page)
    text, outs = dc.attention_module(n, 1, 1, D, pages, page, 1, table.shape[1], "f16", 1.0)
    q, kc, vc = np.zeros((n, 1, D), np.float16), np.zeros((pages, page, 1, D), np.float16), np.ones((pages, page, 1, D), np.float16)
    q[..., 0], kc[table[0, 0], 0, 0, 0] = 1.0, 18.0
    vc[table[0, 0], 0] = 0.0
    mags = {}
    want = decoding.paged_attention(q, kc, vc, table, qs, cl, 1.0, 0, mags)
    assert 1.9e-3 < want.min() and want.max() < 2.1e-3
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl], 256, 1)
    within(got.astype(np.float64), want, dc.split_attention_bound(want, mags, D, "f16"))


@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("dtype, largest", [("f16", 65504.0), ("bf16", float.fromhex("0x1.fep127"))])
def test_paged_attention_of_the_largest_values(gpu_device, n, dtype, largest):
    # their weighted sum stays below them, whatever the weights are before they are divided by their sum
    rng = np.random.default_rng(51)
    H, D, page, B = 2, 32, 16, 5
    new, ctx = [n] * B, [n, n + 3, 150, 700, 2000]
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, page)
    text, outs = dc.attention_module(sum(new), H, H, D, pages, page, B, table.shape[1], dtype, 0.25)
    q, kc = dc.bits(rng.normal(size=(sum(new), H, D)), dtype), dc.bits(rng.normal(size=(pages, page, H, D)), dtype)
    vc = dc.bits(rng.choice([-0.5, 0.25, 0.5, 0.75], (pages, page, H, D)) * largest, dtype)
    vc[..., :4] = dc.bits(np.full(1, 0.75 * largest), dtype)[0]
    mags = {}
    want = decoding.paged_attention(dc.values(q, dtype), dc.values(kc, dtype), dc.values(vc, dtype), table, qs, cl, 0.25, 0, mags)
    (got,) = run(text, outs, [q, kc, vc, table, qs, cl])
    within(dc.values(got, dtype), want, dc.split_attention_bound(want, mags, D, dtype))


# ---- 4-bit products -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("block", [256, 512])
@pytest.mark.parametrize("M, N, K, group, dtype, zeros", [
    (1, 4096, 512, 128, "f16", False), (1, 1, 32, 32, "bf16", True), (2, 100, 96, 32, "f16", True), (3, 1025, 640, 64, "bf16", False), (4, 50, 1280, 256, "f16", True),
    (5, 333, 4096, 32, "bf16", True), (16, 64, 2048, 128, "bf16", False), (17, 40, 384, 64, "f16", False), (70, 33, 256, 128, "f16", True), (130, 20, 1056, 32, "bf16", True),
    (1, 17, 11008, 64, "f16", True), (33, 5000, 160, 32, "f16", False),
    (16, 130, 6144, 64, "f16", True), (9, 50, 8192, 128, "bf16", False), (70, 33, 1056, 32, "bf16", True), (40, 300, 2048, 32, "f16", True)])   # x in slices
def test_matvec_w4(gpu_device, M, N, K, group, dtype, zeros, block):
    rng = np.random.default_rng(19)
    text, outs = dc.w4_module(M, N, K, group, dtype, zeros)
    x, w = dc.bits(rng.normal(size=(M, K)), dtype), rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    s = dc.bits(rng.uniform(-0.02, 0.02, (N, K // group)), dtype)
    z = rng.integers(0, 16, (N, K // group), dtype=np.uint8) if zeros else None
    mags = {}
    want = decoding.matvec_w4(dc.values(x, dtype), w, dc.values(s, dtype), z, mags)
    (got,) = run(text, outs, [x, w, s] + ([z] if zeros else []), block)
    within(dc.values(got, dtype), want, dc.w4_bound(want, mags, K, group, dtype, zeros))


@pytest.mark.parametrize("M, K, group, dtype, zeros, block", [(2, 21760, 32, "f16", False, 512), (2, 21888, 32, "bf16", True, 512), (2, 24576, 128, "f16", True, 256), (3, 16512, 32, "f16", False, 512),
                                                              (64, 896, 32, "bf16", True, 512), (65, 65536, 128, "f16", False, 512), (64, 768, 32, "f16", True, 1024), (128, 11008, 64, "bf16", False, 1024)])
def test_matvec_w4_of_wide_x(gpu_device, M, K, group, dtype, zeros, block):
    rng = np.random.default_rng(48)
    N = 50
    text, outs = dc.w4_module(M, N, K, group, dtype, zeros)
    x, w = dc.bits(rng.normal(size=(M, K)), dtype), rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    s = dc.bits(rng.uniform(-0.02, 0.02, (N, K // group)), dtype)
    z = rng.integers(0, 16, (N, K // group), dtype=np.uint8) if zeros else None
    mags = {}
    want = decoding.matvec_w4(dc.values(x, dtype), w, dc.values(s, dtype), z, mags)
    (got,) = run(text, outs, [x, w, s] + ([z] if zeros else []), block)
    within(dc.values(got, dtype), want, dc.w4_bound(want, mags, K, group, dtype, zeros))


@pytest.mark.parametrize("M, K, group, zeros", [(1, 256, 32, True), (3, 384, 64, True), (2, 512, 128, False), (6, 256, 32, True), (20, 384, 64, True), (9, 512, 256, True), (70, 256, 128, False)])
def test_matvec_w4_of_infinite_x(gpu_device, M, K, group, zeros):
    # f16: a column of a row is infinite; what the definition gives, infinity times value - zero among the rest
    rng = np.random.default_rng(50)
    N = 37
    text, outs = dc.w4_module(M, N, K, group, "f16", zeros)
    x, w = rng.normal(size=(M, K)).astype(np.float16), rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    x[M // 2, rng.integers(K)] = -np.inf
    s = rng.uniform(-0.02, 0.02, (N, K // group)).astype(np.float16)
    z = rng.integers(0, 256, (N, K // group), dtype=np.uint8) if zeros else None
    with np.errstate(invalid="ignore"):
        want = decoding.matvec_w4(x, w, s, z)
    (got,) = run(text, outs, [x, w, s] + ([z] if zeros else []))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    assert np.isinf(got).sum() >= N // 2 and np.isfinite(got).sum() == (M - 1) * N
    finite = np.isfinite(want).all(1)
    mags = {}
    want = decoding.matvec_w4(x[finite], w, s, z, mags)
    if finite.any():
        within(got[finite].astype(np.float64), want, dc.w4_bound(want, mags, K, group, "f16", zeros))


def test_matvec_w4_values_one_by_one(gpu_device):
    # unit rows of x pick single columns: every nibble value at every place of a byte, exactly
    K, N = 128, 16
    for dtype in ("f16", "bf16"):
        text, outs = dc.w4_module(K, N, K, 128, dtype, False)
        w = np.array([[(n + 3 * k) % 16 | ((n * 5 + k) % 16) << 4 for k in range(K // 2)] for n in range(N)], np.uint8)
        (got,) = run(text, outs, [dc.bits(np.eye(K), dtype), w, dc.bits(np.full((N, 1), 0.5), dtype)])
        assert np.array_equal(dc.values(got, dtype), decoding.matvec_w4(np.eye(K), w, np.full((N, 1), 0.5)))


# ---- together -----------------------------------------------------------------------------------------------------------
STEP = dict(L=2, H=128, NH=4, F=256, vocab=300, max_pos=300)


def _run_step(fx, consts, inputs):
    m = MonoNNModule.compile(fx.hlo_text)
    m.set_constants(consts)
    m.load(0)
    out = m.run(inputs, fx.outputs)
    m.close()
    return out


@pytest.mark.parametrize("kw", [
    dict(new_tokens=(1, 1, 1, 1), cached=(100, 37, 200, 5)),
    dict(new_tokens=(50, 3, 1, 0), cached=(0, 5, 9, 20)),
    dict(new_tokens=(1, 1, 1), cached=(100, 37, 0), NKV=2, rotary=True, weights_4bit=32),
    dict(new_tokens=(70, 9), cached=(3, 0), NKV=1, rotary=True, weights_4bit=128, page=8),
])
def test_decoder_step_matches_the_oracle(gpu_device, kw):
    fx = models.gpt2_step(**STEP, **kw)
    consts, inputs = fx.make_constants(21, "random"), fx.make_inputs(21)
    got = _run_step(fx, consts, inputs)
    want = hlo_interp.evaluate(fx.hlo_text, inputs, consts, "fp32")
    for g, w in zip(got, want):
        g, w = g.astype(np.float64), w.astype(np.float64)
        assert np.abs(g - w).max() <= 2e-2 and (g * w).sum() / np.sqrt((g * g).sum() * (w * w).sum()) >= 0.9999


def test_tuned_step_matches_the_oracle(gpu_device, tmp_path):
    from mononn_amd.binding import MonoNNModuleTuner
    fx = models.gpt2_step(**{**STEP, "L": 1}, new_tokens=(1, 20), cached=(70, 9), NKV=2, rotary=True, weights_4bit=32)
    consts, inputs = fx.make_constants(23, "random"), fx.make_inputs(23)
    m = MonoNNModuleTuner.tune(fx.hlo_text, 0, str(tmp_path), budget=2)
    m.set_constants(consts)
    m.load(0)
    got = m.run(inputs, fx.outputs)
    m.close()
    for g, w in zip(got, hlo_interp.evaluate(fx.hlo_text, inputs, consts, "fp32")):
        assert np.abs(g.astype(np.float64) - w.astype(np.float64)).max() <= 2e-2


def test_prompt_in_chunks_then_tokens_equals_the_whole_prompt(gpu_device):
    """Two sequences through the cache -- a chunk, a second chunk, then single tokens, each call on the caches the last
    one left -- give the logits of the dense causal decoder on the same tokens and weights."""
    S, B = 48, 2
    dense = models.gpt2(B=B, S=S, **STEP)
    ids = np.random.default_rng(22).integers(0, STEP["vocab"], (B, S)).astype(np.int32)
    by_role = {dense.constants[n]["role"]: a for n, a in dense.make_constants(22, "random").items()}
    full = MonoNNModule.compile(dense.hlo_text)
    full.set_constants({n: by_role[m["role"]] for n, m in dense.constants.items()})
    full.load(0)
    (want,) = full.run([ids], dense.outputs)
    full.close()
    caches, done = None, 0
    order = None
    for n in (17, 20, 1, 1, 9):
        fx = models.gpt2_step(new_tokens=(n,) * B, cached=(done,) * B, width=4, **STEP)
        inputs = fx.make_inputs(0)
        order = inputs[2] if order is None else order
        assert np.array_equal(order, inputs[2])   # the same pages in every step
        inputs[0] = ids[:, done:done + n].reshape(-1)
        if caches is not None:
            inputs[5:] = caches
        consts = {name: by_role[m["role"]] for name, m in fx.constants.items()}
        logits, *caches = _run_step(fx, consts, inputs)
        w = want[:, done:done + n].reshape(B * n, -1).astype(np.float64)
        assert np.abs(logits.astype(np.float64) - w).max() <= 2e-2
        assert (logits * w).sum() / np.sqrt((logits.astype(np.float64) ** 2).sum() * (w * w).sum()) >= 0.9999
        done += n


# ---- calls ------------------------------------------------------------------------------------------------------------
def _function(text, outs, **kw):
    from mononn_amd.torch_op import MonoNNFunction
    m = MonoNNModule.compile(text)
    m.load(0)
    return MonoNNFunction(m, outs, **kw)


def _attention_call(torch, seed, ctx=(900, 70, 333)):
    rng = np.random.default_rng(seed)
    table, qs, cl, pages = dc.paged_batch(rng, [1, 1, 40], list(ctx), 16)
    text, outs = dc.attention_module(42, 8, 2, 64, pages, 16, 3, table.shape[1], "f16", 0.125)
    a = [rng.normal(size=s).astype(np.float16) for s in ((42, 8, 64), (pages, 16, 2, 64), (pages, 16, 2, 64))] + [table, qs, cl]
    return text, outs, [torch.from_numpy(x).cuda() for x in a]


def test_same_bits_on_every_call_and_on_another_stream(gpu_device):
    import torch
    text, outs, args = _attention_call(torch, 31)
    fn = _function(text, outs, checked=True)
    first = fn(*args)[0].clone()
    for _ in range(20):
        assert torch.equal(fn(*args)[0], first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = fn(*args)[0]
    side.synchronize()
    assert torch.equal(again, first)


def test_captured_and_replayed(gpu_device):
    """A step of append and attention captured once and replayed on new tokens and lengths, with eager work between the
    replays, against the same module called eagerly."""
    import torch
    rng = np.random.default_rng(32)
    new, ctx, page = [1, 1, 1], [200, 90, 17], 16
    table, qs, cl, pages = dc.paged_batch(rng, new, [c + 8 for c in ctx], page)
    D, H, HKV = 64, 4, 2

    def build(e):
        cache = (pages, page, HKV, D)
        q, k, v = e.parameter("f16", (3, H, D), "q"), e.parameter("f16", (3, HKV, D), "k"), e.parameter("f16", (3, HKV, D), "v")
        kc, vc, t = e.parameter("f16", cache, "kc"), e.parameter("f16", cache, "vc"), e.parameter("s32", table.shape, "t")
        s, c, f = e.parameter("s32", (4,), "s"), e.parameter("s32", (3,), "c"), e.parameter("f32", (D // 2,), "f")
        pos = e.parameter("s32", (3,), "positions")
        kc2, vc2 = e.kv_append(k, v, kc, vc, t, s, c, inv_freq=f)
        return [e.paged_attention(e.rope(q, pos, f), kc2, vc2, t, s, c, 0.125), kc2, vc2]
    text, outs = dc.module(build)
    fn = _function(text, outs)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    q, k, v = (dev(rng.normal(size=s).astype(np.float16)) for s in ((3, H, D), (3, HKV, D), (3, HKV, D)))
    kc, vc = (dev(rng.normal(size=(pages, page, HKV, D)).astype(np.float16)) for _ in range(2))
    meta = [dev(table), dev(qs), dev(np.array(ctx, np.int32)), dev(models.rope_frequencies(D)), dev(np.array(ctx, np.int32) - 1)]
    mine = [kc.clone(), vc.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn(q, k, v, kc, vc, *meta)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = fn(q, k, v, kc, vc, *meta)[0]
    kc.copy_(mine[0])
    vc.copy_(mine[1])
    for step in range(5):
        lens = np.array(ctx, np.int32) + step
        for t, shape in ((q, (3, H, D)), (k, (3, HKV, D)), (v, (3, HKV, D))):
            t.copy_(dev(rng.normal(size=shape).astype(np.float16)))
        meta[2].copy_(dev(lens))
        meta[4].copy_(dev(lens - 1))
        graph.replay()
        torch.cuda.synchronize()
        replayed = captured.clone()
        eager = fn(q, k, v, mine[0], mine[1], *meta)[0]
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager) and torch.equal(kc, mine[0]) and torch.equal(vc, mine[1])
    fn.module.synchronize(torch.cuda.current_stream().cuda_stream)


def test_caches_must_be_contiguous_and_of_the_declared_type(gpu_device):
    import torch
    text, outs = dc.append_module(1, 2, 64, 3, 16, 1, 2, "f16")
    fn = _function(text, outs)
    k = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.float16, device="cuda")
    meta = [torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda")]
    with pytest.raises(AssertionError, match="contiguous"):
        fn(k, k, torch.zeros((3, 16, 64, 2), dtype=torch.float16, device="cuda").transpose(2, 3), cache, *meta)
    with pytest.raises(AssertionError, match="declared type"):
        fn(k, k, cache.clone().view(torch.bfloat16), cache, *meta)
    assert not cache.any()


def test_an_updated_input_is_passed_once_and_not_through_the_pure_operator(gpu_device):
    import torch
    from mononn_amd.torch_op import forward
    text, outs = dc.append_module(1, 2, 64, 3, 16, 1, 2, "f16")
    fn = _function(text, outs, checked=True)
    k = torch.ones((1, 2, 64), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((3, 16, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    meta = [torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda")]
    with pytest.raises(AssertionError, match="twice"):
        fn(k, k, kc, kc, *meta)
    with pytest.raises(AssertionError, match="in place"):
        forward(fn, k, k, kc, vc, *meta)
    assert not kc.any() and not vc.any()
    fn(k, k, kc, vc, *meta)   # k and v may be one tensor
    assert kc[0, 0].all() and vc[0, 0].all() and kc.sum() == vc.sum() == 128
    # a cache of another shape is its bytes, as every input is; the result has the declared one and the same storage
    new_k, _ = fn(k, k, kc.view(48, 128), vc, *meta)
    assert new_k.shape == (3, 16, 2, 64) and new_k.data_ptr() == kc.data_ptr()


@pytest.mark.parametrize("returned", [["out"], ["out", "vc"], ["kc", "out"]])
def test_a_cache_that_is_not_returned_is_guarded_too(gpu_device, returned):
    import torch
    from mononn_amd.torch_op import forward
    from test_decoding_operators import append_and_attend
    fn = _function(*append_and_attend(returned), checked=True)
    k = torch.ones((5, 2, 64), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((9, 16, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    strided = torch.zeros((9, 16, 64, 2), dtype=torch.float16, device="cuda").transpose(2, 3)
    meta = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0, 1, 2, 3], [4, 5, 6, 7]], [0, 2, 5], [20, 3])]
    q = torch.ones((5, 4, 64), dtype=torch.float16, device="cuda")
    for caches, words in (((strided, vc), "contiguous"), ((kc, strided), "contiguous"), ((kc.view(torch.bfloat16), vc), "declared type"), ((kc, vc.view(torch.bfloat16)), "declared type"), ((kc, kc), "twice")):
        with pytest.raises(AssertionError, match=words):
            fn(k, k, *caches, *meta, q)
    with pytest.raises(AssertionError, match="in place"):
        forward(fn, k, k, kc, vc, *meta, q)
    torch.cuda.synchronize()
    assert not kc.any() and not vc.any() and not strided.any()
    fn(k, k, kc, vc, *meta, q)
    assert kc.sum() == vc.sum() == 5 * 128 and kc[1, 2].all() and vc[4, :3].all()


@pytest.mark.parametrize("returned", [["out"], ["out", "kc", "vc"]])
def test_autograd_notices_updated_inputs(gpu_device, returned):
    import torch
    from test_decoding_operators import append_and_attend
    fn = _function(*append_and_attend(returned), checked=True)
    k = torch.ones((5, 2, 64), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((9, 16, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    meta = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0, 1, 2, 3], [4, 5, 6, 7]], [0, 2, 5], [20, 3])]
    q = torch.ones((5, 4, 64), dtype=torch.float16, device="cuda")
    leaf = torch.ones((), dtype=torch.float16, device="cuda", requires_grad=True)
    product = (leaf * kc).sum()   # saves kc for its backward pass
    before = [t._version for t in (k, kc, vc, q)]
    fn(k, k, kc, vc, *meta, q)
    assert [t._version for t in (k, kc, vc, q)] == [before[0], before[1] + 1, before[2] + 1, before[3]]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    grows = torch.zeros_like(vc, requires_grad=True)
    with pytest.raises(AssertionError, match="gradient"):
        fn(k, k, kc, grows, *meta, q)
    torch.cuda.synchronize()
    assert not grows.any() and kc._version == before[1] + 1
    with torch.no_grad():
        fn(k, k, kc, grows, *meta, q)
    with torch.inference_mode():
        mine = [torch.zeros_like(kc) for _ in range(2)]
        fn(k, k, *mine, *meta, q)
        assert torch.equal(mine[0], kc) and torch.equal(mine[1], grows)


def test_two_functions_in_two_graphs(gpu_device):
    """Parts of split sequences lie in each function's own memory: graphs of two, replayed in turn, keep their results."""
    import torch
    made = []
    for seed, ctx in ((41, (3000, 70, 900)), (42, (50, 2000, 400))):
        text, outs, args = _attention_call(torch, seed, ctx)
        fn = _function(text, outs)
        want = fn(*args)[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn(*args)[0]
        made.append((fn, args, want, graph, out))
    for i in range(6):
        for fn, args, want, graph, out in made:
            out.zero_()
            graph.replay()
            if i % 2:
                assert torch.equal(fn(*args)[0], want)
        torch.cuda.synchronize()
        for *_, want, graph, out in made:
            assert torch.equal(out, want)


def test_inputs_that_are_views(gpu_device):
    import torch
    text, outs, args = _attention_call(torch, 43)
    fn = _function(text, outs, checked=True)
    want = fn(*args)[0]
    q = torch.zeros((42, 8, 2, 64), dtype=torch.float16, device="cuda")
    q[:, :, 1] = args[0]
    assert torch.equal(fn(q[:, :, 1], *args[1:])[0], want)
    flat = torch.zeros(args[0].numel() + 8, dtype=torch.float16, device="cuda")
    flat[8:] = args[0].reshape(-1)
    assert torch.equal(fn(flat[8:].view(args[0].shape), *args[1:])[0], want)
    with pytest.raises(AssertionError, match="aligned"):
        fn(flat[1:-7].view(args[0].shape), *args[1:])


def test_launch_with_the_static_arena_and_null_slots(gpu_device):
    import torch
    from mononn_amd import MonoNNError
    text, outs, args = _attention_call(torch, 44)
    (want,) = _function(text, outs, checked=True)(*args)
    m = MonoNNModule.compile(text)
    m.load(0)
    assert 0 < m.buffer_info()["temp"]
    out = torch.empty_like(want)
    stream = torch.cuda.current_stream().cuda_stream
    from mononn_amd import binding
    if m.buffer_info()["temp"] <= binding._lib.mononn_static_temp_bytes():
        m.launch_static_temp([t.data_ptr() for t in args] + [out.data_ptr()], stream)
        m.synchronize(stream)
        assert torch.equal(out, want)
    with pytest.raises(MonoNNError):
        m.launch_static_temp([t.data_ptr() for t in args] + [0], stream)
    m.close()
    text, outs = dc.append_module(1, 2, 64, 3, 16, 1, 2, "f16")
    a = MonoNNModule.compile(text)
    a.load(0)
    k = torch.ones((1, 2, 64), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((3, 16, 2, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    meta = [torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda")]
    a.launch_static_temp([t.data_ptr() for t in (k, k, kc, vc, *meta)] + [0, 0], stream)   # the live-outs are the caches: no buffers of their own
    a.synchronize(stream)
    assert kc.sum() == vc.sum() == 128
    with pytest.raises(MonoNNError):
        a.launch_static_temp([k.data_ptr(), k.data_ptr(), 0, vc.data_ptr()] + [t.data_ptr() for t in meta] + [0, 0], stream)
    a.close()


@pytest.mark.parametrize("new, ctx, H, HKV, D", [([1] * 32, [40 + 61 * i for i in range(32)], 32, 8, 128), ([300, 1, 40], [300, 999, 70], 32, 8, 128), ([1] * 90, [200] * 90, 32, 8, 128), ([2, 2], [500, 60], 8, 1, 256)])
def test_attention_launches_with_the_static_arena(gpu_device, new, ctx, H, HKV, D):
    import torch
    from mononn_amd import binding
    rng = np.random.default_rng(49)
    table, qs, cl, pages = dc.paged_batch(rng, new, ctx, 16)
    text, outs = dc.attention_module(sum(new), H, HKV, D, pages, 16, len(new), table.shape[1], "bf16", D ** -0.5)
    args = [torch.from_numpy(rng.normal(size=s).astype(np.float32)).cuda().bfloat16() for s in ((sum(new), H, D), (pages, 16, HKV, D), (pages, 16, HKV, D))]
    args += [torch.from_numpy(a).cuda() for a in (table, qs, cl)]
    m = MonoNNModule.compile(text)
    m.load(0)
    assert m.buffer_info()["temp"] <= binding._lib.mononn_static_temp_bytes()
    from mononn_amd.torch_op import MonoNNFunction
    (want,) = MonoNNFunction(m, outs, checked=True)(*args)
    out = torch.zeros_like(want)
    stream = torch.cuda.current_stream().cuda_stream
    m.launch_static_temp([t.data_ptr() for t in args] + [out.data_ptr()], stream)
    m.synchronize(stream)
    assert torch.equal(out, want) and out.any()
    m.close()


def test_operands_and_results_in_other_layouts(gpu_device):
    # any order of dimensions in memory at the module's boundary; the operators themselves work on row-major values
    rng = np.random.default_rng(45)
    T, H, HKV, D, page = 5, 4, 2, 32, 4
    table, qs, cl, pages = dc.paged_batch(rng, [2, 3], [9, 30], page)
    text, outs = dc.attention_module(T, H, HKV, D, pages, page, 2, table.shape[1], "f16", 0.2)
    args = [rng.normal(size=s).astype(np.float16) for s in ((T, H, D), (pages, page, HKV, D), (pages, page, HKV, D))] + [table, qs, cl]
    (want,) = run(text, outs, args)
    # q with the heads slowest, the keys with the elements slowest, the table by columns
    q, c, t = f"f16[{T},{H},{D}]", f"f16[{pages},{page},{HKV},{D}]", f"s32[2,{table.shape[1]}]"
    turned = [args[0].transpose(1, 0, 2), args[1].transpose(3, 2, 1, 0), args[2], table.T, qs, cl]
    lines = []
    for line in text.splitlines():
        if "parameter(0)" in line:
            line = line.replace(q + "{2,1,0}", q + "{2,0,1}")
        elif "parameter(1)" in line:
            line = line.replace(c + "{3,2,1,0}", c + "{0,1,2,3}")
        elif "parameter(3)" in line:
            line = line.replace(t + "{1,0}", t + "{0,1}")
        lines.append(line)
    assert lines != text.splitlines()
    (got,) = run("\n".join(lines), outs, [np.ascontiguousarray(a) for a in turned])
    assert np.array_equal(got, want)


def test_weights_as_constants(gpu_device):
    # the usual home of weights: module constants, uploaded once, read in place
    rng = np.random.default_rng(33)
    names = {}

    def build(e):
        w, s = e.elided_constant("u8", (70, 128), "proj/weight_4bit"), e.elided_constant("f16", (70, 4), "proj/scales")
        names.update(w=w.name, s=s.name)
        return e.matvec_w4(e.parameter("f16", (3, 256), "x"), w, s)
    text, outs = dc.module(build)
    x, w, s = rng.normal(size=(3, 256)).astype(np.float16), rng.integers(0, 256, (70, 128), dtype=np.uint8), rng.uniform(0.001, 0.02, (70, 4)).astype(np.float16)
    m = MonoNNModule.compile(text)
    m.set_constants({names["w"]: w, names["s"]: s})
    m.load(0)
    (got,) = m.run([x], outs)
    mags = {}
    want = decoding.matvec_w4(x, w, s, None, mags)
    within(got.astype(np.float64), want, dc.w4_bound(want, mags, 256, 64, "f16", False))
    m.close()
