"""The key/value cache's kernels against their definitions in 64 bits.

Tolerances: keys that become four bits are rounded once from rotated values that
are exact to about 2^-50, so pages must hold the very codes of the 64-bit result,
and so must values, which are not rotated. Rows that become bf16 or stay fp32 are
rotated in fp32: r = a cos - b sin with cos, sin and one product rounded and the
fused sum rounded is off by 2^-24 (|a cos| + 2 |b sin| + |r|), at most 2^-24 * 3
(|a| + |b|), which comes to the half step of the type. Attention is bounded
element by element (kv_model.attention)."""

import ctypes

import numpy as np
import pytest

import awa_hip as A
import kv_model as M

pytestmark = pytest.mark.gpu


def new_rows(rng, counts, heads, dim, dtype, std=1.0):
    return M.as_type(rng.standard_normal((sum(counts), heads, dim)) * std, dtype)


def rotation_bound(x, want, rope_dim, axes=1, halves=False, dtype="f32", **_):
    """How far a row rotated in fp32 and stored as dtype may be from `want`."""
    a = np.abs(np.asarray(x, np.float64))
    both = np.zeros_like(a)
    lo, hi = ((slice(0, rope_dim // 2), slice(rope_dim // 2, rope_dim)) if halves
              else (slice(0, rope_dim, 2), slice(1, rope_dim, 2)))
    both[..., lo] = both[..., hi] = a[..., lo] + a[..., hi]
    fp32 = 3.0 * 2.0 ** -24 * both
    return fp32 + (M.HALF[dtype] * (np.abs(want) + fp32) if dtype == "bf16" else 0.0)


def expected_pools(cache, counts, k, v, skip=()):
    """The pools after appending k and v (64 bits), sequence by sequence."""
    pools = {n: x.copy() for n, x in cache.host.items()}
    at = 0
    for s, n in enumerate(counts):
        length = int(cache.lengths[s])
        for j in range(n):
            slot = length - n + j
            page = cache.table[s, slot // cache.page]
            if s in skip or not 0 <= page < cache.pages:
                continue
            for name, x in (("k", k), ("v", v)):
                if cache.four:
                    codes, byte = M.encode4(x[at + j])
                    pools[name][page, :, slot % cache.page] = codes
                    pools[name + "_scale"][page, :, slot % cache.page] = byte
                else:
                    # Rounded from 64 bits: through fp32 only where that is exact.
                    pools[name][page, :, slot % cache.page] = bf16_bits64(x[at + j])
        at += n
    return pools


def bf16_bits64(x):
    """x (64 bits) to the nearest bf16, ties to even, without a first rounding to fp32."""
    x = np.asarray(x, np.float64)
    f = x.astype(np.float32)
    back = f.astype(np.float64)
    bits = f.view(np.uint32)
    away = np.abs(back) < np.abs(x)
    odd = np.where((back != x) & (bits & 1 == 0) & np.isfinite(x), np.where(away, bits + 1, bits - 1), bits)
    return A.f32_to_bf16_bits(odd.astype(np.uint32).view(np.float32))


def check_pools(cache, want, counts=None, k=None, rope=None):
    """The pools; of bf16 pages the appended keys (k before the rotation) within
    their bound, and all else to the bit."""
    got = cache.download()
    if not cache.four and rope is not None:
        at = 0
        for s, n in enumerate(counts):
            for j in range(n):
                slot = int(cache.lengths[s]) - n + j
                where = (cache.table[s, slot // cache.page], slice(None), slot % cache.page)
                g, w = (A.bf16_bits_to_f32(x["k"][where]).astype(np.float64) for x in (got, want))
                exact = rope["rows"][at + j]
                assert (np.abs(g - exact) <= rotation_bound(k[at + j], exact, dtype="bf16", **rope["kw"])).all()
                got["k"][where] = want["k"][where]
            at += n
    for name, x in want.items():
        bad = np.argwhere(got[name] != x)
        assert len(bad) == 0, f"{name}: {len(bad)} of {x.size} differ, first at {bad[:3].tolist()}"


ROPES = {"neighbours": dict(rope_dim=64, axes=1), "halves": dict(rope_dim=64, axes=1, halves=True),
         "part_halves": dict(rope_dim=32, axes=1, halves=True), "three_axes": dict(rope_dim=60, axes=3),
         "few": dict(rope_dim=2, axes=1), "none": None}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("rope", list(ROPES))
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(128, 4, 2, 16), (64, 3, 3, 64)])
def test_append(gpu, dtype, fmt, rope, dim, heads, kv_heads, page):
    rng = np.random.default_rng(3)
    counts, before = [5, 0, 1, 18, 33], [0, 4, 40, 15, 100]
    cache = M.Cache(fmt, [n + b for n, b in zip(counts, before)], kv_heads, dim, page, stride=20)
    desc = cache.upload()
    total = sum(counts) + 3  # three rows behind the last sequence's
    wide = (heads + 2 * kv_heads) * dim
    q, k, v = (new_rows(rng, [total], h, dim, dtype) for h in (heads, kv_heads, kv_heads))
    # Views of one projection [token][q heads, k heads, v heads].
    qd = M.Rows(q, dtype, wide, 0)
    kd, vd = M.Rows(k, dtype, wide, heads * dim), M.Rows(v, dtype, wide + 16, 8)
    out = M.Rows(np.full(q.shape, 5.0), dtype, heads * dim + 24, 16)
    cu = M.ints(np.cumsum([0] + counts))
    kw = ROPES[rope]
    if kw is None:
        A.kv_append(desc, A.KvRows(40, cu.ptr), kd.blob, vd.blob)
        kr = k.astype(np.float64)
    else:
        if dim == 128:
            kw = dict(kw, rope_dim=kw["rope_dim"] * 2)
        r = A.Rope(**kw)
        pos = rng.integers(0, 2000, (total, kw["axes"]))
        A.kv_append(desc, A.KvRows(40, cu.ptr), kd.blob, vd.blob, r, M_keep(pos), qd.blob, out.blob)
        kr = M.rotate(k, pos, **kw)
    A.synchronize()
    check_pools(cache, expected_pools(cache, counts, kr, v.astype(np.float64)), counts, k,
                kw and {"rows": kr, "kw": kw})
    assert cache.status() == 0
    if kw is not None:
        got, want = out.read(), M.rotate(q, pos, **kw)
        n = sum(counts)
        assert (np.abs(got[:n] - want[:n]) <= rotation_bound(q, want, dtype=dtype, **kw)[:n]).all()
        assert (got[n:] == 5.0).all()
        whole = out.read(whole=True)
        assert (whole[:, :16] == 7.0).all() and (whole[:, 16 + heads * dim:] == 7.0).all()


_kept = []


def M_keep(x):
    """Device copy of positions that lives until the test process ends."""
    _kept.append(M.ints(x))
    return _kept[-1].ptr


@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
def test_append_far_positions(gpu, fmt):
    """Positions up to both ends of 32 bits, and the slots where none are given."""
    rng = np.random.default_rng(4)
    pos = np.array([[0], [1], [-1], [2 ** 31 - 1], [-2 ** 31], [1 << 20], [123456789], [-987654321]])
    cache = M.Cache(fmt, [len(pos)], 2, 128, 16)
    desc = cache.upload()
    k, v = (new_rows(rng, [len(pos)], 2, 128, "f32") for _ in range(2))
    q = new_rows(rng, [len(pos)], 2, 128, "f32")
    kd, vd, qd = (M.Rows(x, "f32") for x in (k, v, q))
    A.kv_append(desc, A.KvRows(len(pos)), kd.blob, vd.blob, A.Rope(128), M_keep(pos), qd.blob, qd.blob)  # in place
    want = M.rotate(q, pos, 128)
    # 2^31 positions of an angle that is exact to 2^-64 of a turn each.
    assert (np.abs(qd.read() - want) <= rotation_bound(q, want, 128) + 2 * np.pi * 2.0 ** -33 * 2 * np.abs(q).max()).all()

    cache = M.Cache(fmt, [70], 2, 128, 16)
    desc = cache.upload()
    A.kv_append(desc, A.KvRows(len(pos)), kd.blob, vd.blob, A.Rope(126))
    kr = M.rotate(k, np.arange(62, 70)[:, None], 126)
    check_pools(cache, expected_pools(cache, [8], kr, v.astype(np.float64)), [8], k,
                {"rows": kr, "kw": {"rope_dim": 126}})


def test_append_given_frequencies(gpu):
    rng = np.random.default_rng(5)
    f = [3.0, -0.5, 0.0, 1e-3, 2.5, 1e-7, 7.0, 0.125]
    cache = M.Cache("4bit", [9], 1, 64, 16)
    desc = cache.upload()
    k, v = (new_rows(rng, [9], 1, 64, "bf16") for _ in range(2))
    pos = rng.integers(-500, 500, (9, 1))
    A.kv_append(desc, A.KvRows(9), M.Rows(k, "bf16").blob, M.Rows(v, "bf16").blob,
                A.Rope(16, frequencies=f, halves=True), M_keep(pos))
    A.synchronize()
    check_pools(cache, expected_pools(cache, [9], M.rotate(k, pos, 16, halves=True, frequencies=f),
                                      v.astype(np.float64)))


def test_append_turns_as_mmrope(gpu):
    """The block's own rotation (three axes, 126 features): awa_mmrope's fp32
    angles are off by half a step of at most 128, its products by 2^-23."""
    plan = A.Plan(A.LayerParams(2, 4, 4, 1, 1, 1, 5, False))
    plan.upload()
    rows = plan.info.sequence_tokens
    rng = np.random.default_rng(6)
    x = rng.standard_normal((rows, 3, 1, 128)).astype(np.float32)
    src, dst = M.Rows(x.reshape(rows, 3, 128), "f32"), M.Rows(np.zeros((rows, 3, 128)), "f32")
    plan.mmrope(src.blob, dst.blob)
    t, h, w = np.meshgrid(np.arange(2), np.arange(4), np.arange(4), indexing="ij")
    video = np.stack([t.ravel() + 5, h.ravel(), w.ravel()], 1)
    pos = np.concatenate([video, np.repeat(np.arange(5)[:, None], 3, 1)])
    assert len(pos) == rows
    q, out = M.Rows(x[:, 0], "f32"), M.Rows(np.zeros((rows, 1, 128)), "f32")
    cache = M.Cache("bf16", [rows], 1, 128, 16)
    A.kv_append(cache.upload(), A.KvRows(rows), M.Rows(x[:, 1], "f32").blob, M.Rows(x[:, 2], "f32").blob,
                A.Rope(126, 3), M_keep(pos), q.blob, out.blob)
    A.synchronize()
    index = plan.sequence_index()
    assert (np.sort(index) == np.arange(rows)).all()
    np.testing.assert_allclose(out.read()[index, 0], dst.read()[:, 0], atol=4e-6 * 4)


def test_append_four_bits_of_all_kinds(gpu):
    """Zeros, ties, values of every magnitude, NaN and infinities: other groups are not touched by them."""
    rng = np.random.default_rng(7)
    x = np.zeros((16, 1, 128), np.float32)
    x[1, 0, :8] = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x[2] = -x[1]
    x[3, 0, 3], x[3, 0, 40], x[3, 0, 99] = np.nan, np.inf, -np.inf
    x[4] = rng.standard_normal(128) * 3e38 / 4
    x[5] = rng.standard_normal(128) * 1e-37
    x[6, 0, 0] = np.finfo(np.float32).max
    x[7, 0, 31], x[7, 0, 32] = 7.0, np.nextafter(np.float32(7.0), np.float32(8.0))
    x[8:] = rng.standard_normal((8, 1, 128)) * np.exp2(rng.integers(-60, 60, (8, 1, 128)))
    cache = M.Cache("4bit", [16], 1, 128, 16)
    desc = cache.upload()
    rows = M.Rows(x, "f32")
    A.kv_append(desc, A.KvRows(16), rows.blob, rows.blob)
    A.synchronize()
    check_pools(cache, expected_pools(cache, [16], x.astype(np.float64), x.astype(np.float64)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("dim", [64, 128])
def test_read(gpu, dtype, fmt, dim):
    counts, lengths = [40, 0, 17, 3], [40, 9, 90, 100]
    cache = M.Cache(fmt, lengths, 3, dim, 32)
    if fmt == "4bit":
        cache.host["k_scale"][0] = 255
        cache.host["v_scale"][1, :, ::3] = 100
    desc = cache.upload()
    total = sum(counts) + 2
    k, v = (M.Rows(np.full((total, 3, dim), 5.0), dtype, 3 * dim + 32, 16) for _ in range(2))
    A.kv_read(desc, A.KvRows(40, M_keep(np.cumsum([0] + counts))), k.blob, v.blob)
    A.synchronize()
    for name, got in (("k", k.read()), ("v", v.read())):
        at = 0
        for s, n in enumerate(counts):
            np.testing.assert_array_equal(got[at:at + n], cache.rows(name, s)[0][lengths[s] - n:])
            at += n
        assert (got[at:] == 5.0).all()
    assert cache.status() == 0


def test_many_rows_and_sequences(gpu):
    """Whole tokens a workgroup (many rows), and more sequences than a wave has lanes."""
    rng = np.random.default_rng(8)
    counts = [int(n) for n in rng.integers(0, 40, 150)]
    lengths = [n + int(b) for n, b in zip(counts, rng.integers(0, 60, 150))]
    for fmt in ("bf16", "4bit"):
        cache = M.Cache(fmt, lengths, 2, 64, 16)
        desc = cache.upload()
        total = sum(counts) + 1
        assert total > 2048
        k, v = (new_rows(rng, [total], 2, 64, "bf16") for _ in range(2))
        rows = A.KvRows(40, M_keep(np.cumsum([0] + counts)))
        A.kv_append(desc, rows, M.Rows(k, "bf16").blob, M.Rows(v, "bf16").blob)
        A.synchronize()
        want = expected_pools(cache, counts, k.astype(np.float64), v.astype(np.float64))
        check_pools(cache, want)
        cache.host = want
        ko, vo = (M.Rows(np.full(k.shape, 5.0), "f32") for _ in range(2))
        A.kv_read(desc, rows, ko.blob, vo.blob)
        A.synchronize()
        at = 0
        for s, n in enumerate(counts):
            np.testing.assert_array_equal(vo.read()[at:at + n], cache.rows("v", s)[0][lengths[s] - n:])
            at += n
        assert (ko.read()[at:] == 5.0).all()


@pytest.mark.parametrize("n", [65, 4097])
@pytest.mark.parametrize("order", ["kept", "broken"])
def test_rows_of_thousands_of_sequences(gpu, n, order):
    """Every row finds its sequence, beside empty ones; of cu_rows out of order all
    rows that one sequence alone claims."""
    rng = np.random.default_rng(12)
    counts = [int(c) for c in rng.choice([0, 1, 1, 1, 2], n)]
    cu = np.cumsum([0] + counts)
    total = int(cu[-1]) + 3
    if order == "broken":
        cu[n // 2] = 0  # one sequence ends before it begins, the next has too many rows
    cache = M.Cache("bf16", [c + 1 for c in counts], 1, 64, 16)
    desc = cache.upload()
    x = new_rows(rng, [total], 1, 64, "bf16")
    A.kv_append(desc, A.KvRows(2, M_keep(cu)), M.Rows(x, "bf16").blob, M.Rows(x, "bf16").blob)
    A.synchronize()
    assert cache.status() == (A.KV_BAD_ROWS if order == "broken" else 0)
    want = cache.host["v"].copy()
    for s in range(n):
        rows = int(cu[s + 1]) - int(cu[s])
        if not 0 <= rows <= 2:
            continue
        for j in range(rows):
            slot = int(cache.lengths[s]) - rows + j
            want[cache.table[s, slot // 16], 0, slot % 16] = A.f32_to_bf16_bits(x[cu[s] + j, 0])
    np.testing.assert_array_equal(cache.download()["v"], want)


def test_what_does_not_fit_is_left_out_and_told(gpu):
    """Bad pages, lengths and rows: told in the status, nothing read or written for them."""
    rng = np.random.default_rng(9)
    counts = [4, 4, 4, 4]
    for bad, status in [({"page": (1, 2, -1)}, A.KV_BAD_PAGE), ({"page": (1, 2, 10 ** 6)}, A.KV_BAD_PAGE),
                        ({"length": (2, -5)}, A.KV_BAD_LENGTH), ({"length": (2, 3)}, A.KV_BAD_LENGTH),
                        ({"length": (2, 16 * 3 + 1)}, A.KV_BAD_LENGTH), ({"cu": [0, 4, 12, 12, 16]}, A.KV_BAD_ROWS),
                        ({"cu": [0, 4, 8, 12, 17]}, A.KV_BAD_ROWS), ({"cu": [0, 4, 2, 12, 16]}, A.KV_BAD_ROWS)]:
        cache = M.Cache("bf16", [20, 40, 36, 4], 1, 64, 16)
        desc = cache.upload()
        cu = [0, 4, 8, 12, 16]
        if "page" in bad:
            s, i, p = bad["page"]
            cache.table[s, i] = p
            cache.set(table=cache.table)
        if "length" in bad:
            cache.lengths[bad["length"][0]] = bad["length"][1]
            cache.set(lengths=cache.lengths)
        cu = bad.get("cu", cu)
        rows = A.KvRows(4, M_keep(cu))
        x = new_rows(rng, counts, 1, 64, "bf16")
        blob, ko, vo, out = (M.Rows(y, "bf16") for y in (x, x * 0 + 5, x * 0 + 5, x * 0 + 5))
        q = M.Rows(x, "bf16")
        qo = M.Rows(x * 0 + 5, "bf16")
        A.kv_append(desc, rows, blob.blob, blob.blob, A.Rope(64), None, q.blob, qo.blob)
        A.synchronize()
        assert cache.status() == status, bad
        pools = cache.download()
        good = []
        for s in range(4):
            a, b = cu[s], cu[s + 1]
            n = b - a
            length = int(cache.lengths[s])
            if a < 0 or n < 0 or n > 4 or b > 16 or not n <= length <= 48:
                continue
            good.append((s, a, n, length))
        touched = np.zeros((cache.pages, 16), bool)
        for s, a, n, length in good:
            for j in range(n):
                slot = length - n + j
                page = cache.table[s, slot // 16]
                if 0 <= page < cache.pages:
                    touched[page, slot % 16] = True
                    np.testing.assert_array_equal(pools["v"][page, 0, slot % 16], A.f32_to_bf16_bits(x[a + j, 0]))
        for name in ("k", "v"):
            same = (pools[name] == cache.host[name])[:, 0].all(-1)
            assert (same | touched).all()
        cache.dev["status"].zero()
        cache.host = pools
        A.kv_read(desc, rows, ko.blob, vo.blob)
        n = A.kv_attention_workspace(desc, rows, q.blob, A.KvMask())
        ws = A.DeviceBuffer(max(n, 16))
        A.kv_attention(desc, rows, q.blob, A.KvMask(), 0.125, out.blob, ws.ptr, n)
        A.synchronize()
        assert cache.status() == status, bad
        want_v = np.full(x.shape, 5.0)
        want = np.full(x.shape, 5.0)
        bound = np.zeros(x.shape)
        for s, a, n, length in good:
            v, ok = cache.rows("v", s)
            k, _ = cache.rows("k", s)
            for j in range(n):
                if ok[length - n + j]:
                    want_v[a + j] = v[length - n + j]
            want[a:a + n], bound[a:a + n] = M.attention(x[a:a + n], k, v, length, 0, 0, 1, 0.125, "bf16", ok)
        np.testing.assert_array_equal(vo.read(), want_v)
        assert (np.abs(out.read() - want) <= bound).all(), bad


# ---- attention ----

def run_attention(cache, counts, q, dtype, window=0, sinks=0, block=1, scale=None, max_length=0, spare=0, stream=None,
                  pitch=0):
    scale = cache.dim ** -0.5 if scale is None else scale
    qd = M.Rows(q, dtype, pitch, 8 if pitch else 0)
    out = M.Rows(np.full(q.shape, 5.0), dtype, pitch, 16 if pitch else 0)
    mask = A.KvMask(window, sinks, block, max_length)
    rows = A.KvRows(max(max(counts), 1), M_keep(np.cumsum([0] + counts)))
    n = A.kv_attention_workspace(cache.desc, rows, qd.blob, mask)
    ws = A.DeviceBuffer(max(n, 16))
    A.kv_attention(cache.desc, rows, qd.blob, mask, scale, out.blob, ws.ptr, n, stream)
    A.synchronize(stream)
    got = out.read()
    assert (got[sum(counts):] == 5.0).all()  # rows behind the last sequence's
    return got


def check_attention(cache, counts, q, dtype, got, window=0, sinks=0, block=1, scale=None, sequences=None):
    scale = cache.dim ** -0.5 if scale is None else scale
    at = 0
    for s, n in enumerate(counts):
        if sequences is None or s in sequences:
            k, ok = cache.rows("k", s)
            v, _ = cache.rows("v", s)
            want, bound = M.attention(q[at:at + n], k, v, int(cache.lengths[s]), window, sinks, block, scale, dtype, ok)
            with np.errstate(invalid="ignore"):
                off = np.abs(got[at:at + n] - want)
            same = (np.isnan(got[at:at + n]) & np.isnan(want)) | (got[at:at + n] == want)
            bad = ~(same | (off <= bound))
            assert not bad.any(), (s, np.argwhere(bad)[:4].tolist(), float(np.nanmax(off)), float(np.nanmax(bound)))
        at += n


CASES = [
    # counts, lengths, heads, kv heads, page, window, sinks, block
    ([1], [1], 2, 2, 16, 0, 0, 1),
    ([1, 1, 1], [700, 33, 1], 4, 2, 16, 0, 0, 1),
    ([1, 0, 1, 1], [129, 64, 65, 2000], 5, 1, 64, 100, 4, 1),
    ([3, 1, 4], [300, 17, 4], 8, 2, 32, 0, 0, 1),
    ([4, 2], [500, 90], 6, 6, 16, 37, 5, 1),
    ([17, 1, 60], [17, 400, 333], 4, 4, 16, 0, 0, 1),
    ([130, 5], [400, 5], 2, 1, 128, 64, 3, 1),
    ([64, 16], [84, 52], 2, 2, 16, 0, 4, 16),
    ([100], [250], 3, 3, 16, 48, 10, 24),
    ([90, 200], [91, 331], 6, 2, 16, 1, 0, 1),
    ([33], [800], 2, 2, 16, 200, 300, 1),
    ([300, 257], [300, 1000], 2, 2, 256, 0, 0, 1),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(gpu, dtype, fmt, dim, case):
    counts, lengths, heads, kv_heads, page, window, sinks, block = CASES[case]
    rng = np.random.default_rng(10 + case)
    cache = M.Cache(fmt, lengths, kv_heads, dim, page, seed=case)
    cache.upload()
    q = new_rows(rng, [sum(counts) + 2], heads, dim, dtype, std=2.0)
    got = run_attention(cache, counts, q, dtype, window, sinks, block, pitch=heads * dim + 24)
    check_attention(cache, counts, q, dtype, got, window, sinks, block)
    assert cache.status() == 0
    # The bound of the lengths sets the split alone.
    short = run_attention(cache, counts, q, dtype, window, sinks, block, max_length=max(lengths))
    check_attention(cache, counts, q, dtype, short, window, sinks, block)


MIXED = [
    # counts, lengths, heads, kv heads, window, sinks, bounds of the lengths
    ([1, 200, 0, 3, 43, 42, 70], [5000, 300, 10, 2100, 90, 1500, 2000], 6, 2, 0, 0, (0, 5000, 5)),
    ([128, 129, 1], [700, 700, 3000], 2, 2, 1100, 7, (0, 3000, 64)),
    ([1, 2, 300], [9000, 2, 301], 4, 1, 0, 0, (0, 9000, 300)),
    ([12, 1, 9], [800, 3000, 9], 4, 1, 0, 0, (0, 3000, 1)),
    ([1, 2, 1], [400, 1300, 1], 140, 1, 0, 0, (0, 1300, 70)),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("case", range(len(MIXED)))
def test_single_tokens_beside_chunks(gpu, dtype, fmt, case):
    """Sequences of few rows are dealt out otherwise than long ones of the same
    call; a bound of the lengths that they pass changes only the split."""
    counts, lengths, heads, kv_heads, window, sinks, bounds = MIXED[case]
    rng = np.random.default_rng(40 + case)
    cache = M.Cache(fmt, lengths, kv_heads, 64, 32, seed=case)
    cache.upload()
    q = new_rows(rng, [sum(counts) + 2], heads, 64, dtype, std=2.0)
    for bound in bounds:
        got = run_attention(cache, counts, q, dtype, window, sinks, max_length=bound)
        check_attention(cache, counts, q, dtype, got, window, sinks)
    assert cache.status() == 0


@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
def test_many_single_tokens_beside_a_chunk(gpu, fmt):
    """Parts numbered through over sequences of 0, 1, a few and many rows, some of
    which do not fit together: more than a wave's and more than a workgroup's."""
    rng = np.random.default_rng(47)
    for n, most, heads, kv_heads in ((100, 700, 8, 4), (1500, 300, 2, 1), (70, 900, 6, 2)):
        counts = [1] * n
        for s, x in ((0, 0), (1, 40), (n // 2, most), (n - 3, 129), (n - 2, 0), (n - 1, 3)):
            counts[s] = x
        lengths = [int(x) + c for x, c in zip(rng.integers(0, 60, n), counts)]
        lengths[2], lengths[n // 2 + 1] = 3000, 1500
        cache = M.Cache(fmt, lengths, kv_heads, 64, 16)
        cache.lengths[5] = 0                      # below its new rows
        cache.lengths[6] = cache.table.shape[1] * 16 + 1
        cache.upload()
        q = new_rows(rng, [sum(counts) + 1], heads, 64, "bf16", std=2.0)
        for bound in (0, 3000):
            got = run_attention(cache, counts, q, "bf16", max_length=bound)
            check_attention(cache, counts, q, "bf16", got, sequences=set(range(n)) - {5, 6})
            for s in (5, 6):
                assert (got[sum(counts[:s])] == 5.0).all()
        assert cache.status() == A.KV_BAD_LENGTH


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("4bit", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,window", [
    ([2150], [5500], 64, 64, 0), ([1500], [5500], 96, 32, 0), ([1700], [4500], 64, 64, 2100),
    ([600, 480], [2700, 2500], 120, 40, 0)])
def test_first_tiles_of_a_chunk_split(gpu, fmt, dtype, counts, lengths, heads, kv_heads, window):
    """Somewhat more row tiles than the device takes at a time: the first ones, which
    come last, are split. Rows beside every border of tiles, and others."""
    dim, rng = 64, np.random.default_rng(49)
    cache = M.Cache(fmt, lengths, kv_heads, dim, 64)
    cache.upload()
    q = new_rows(rng, [sum(counts)], heads, dim, dtype, std=2.0)
    got = run_attention(cache, counts, q, dtype, window, 5, max_length=max(lengths))
    again = run_attention(cache, counts, q, dtype, window, 5, max_length=max(lengths) // 2)
    group, at = heads // kv_heads, 0
    for s, n in enumerate(counts):
        k, _ = cache.rows("k", s)
        v, _ = cache.rows("v", s)
        borders = {t * 128 // group + d for t in range(n * group // 128 + 1) for d in (-1, 0)}
        for j in sorted({j for j in borders if 0 <= j < n} | {0, n - 1} | {int(x) for x in rng.integers(0, n, 20)}):
            h = int(rng.integers(0, kv_heads))
            end = lengths[s] - n + j + 1
            want, bound = M.attention(q[at + j:at + j + 1, h * group:(h + 1) * group], k[:end, h:h + 1], v[:end, h:h + 1],
                                      end, window, 5, 1, dim ** -0.5, dtype)
            for x in (got, again):
                assert (np.abs(x[at + j, h * group:(h + 1) * group] - want[0]) <= bound[0]).all(), (s, j, h)
        at += n
    assert cache.status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 33)])
def test_about_a_workgroup_a_cu(gpu, dtype, fmt, dim, window, sinks):
    """Single and draft tokens of a batch whose heads are about as many as CUs."""
    rng = np.random.default_rng(51)
    counts = [int(x) for x in rng.choice([0, 1, 1, 2], 60)]
    lengths = [c + int(x) for c, x in zip(counts, rng.integers(0, 1200, 60))]
    cache = M.Cache(fmt, lengths, 2, dim, 32)
    cache.upload()
    q = new_rows(rng, [sum(counts)], 4, dim, dtype, std=2.0)
    for bound in (max(lengths), 1100):
        got = run_attention(cache, counts, q, dtype, window, sinks, max_length=bound)
        check_attention(cache, counts, q, dtype, got, window, sinks)
    assert cache.status() == 0


def test_rows_bounds_above_the_rows(gpu):
    """max_rows as a bound: sequences may all be shorter."""
    rng = np.random.default_rng(46)
    for counts, lengths, most in (([1, 2], [3000, 700], 500), ([3], [2000], 1000), ([150, 1], [160, 2500], 151)):
        cache = M.Cache("bf16", lengths, 1, 64, 16)
        cache.upload()
        q = new_rows(rng, counts, 4, 64, "bf16")
        qd, out = M.Rows(q, "bf16"), M.Rows(np.full(q.shape, 5.0), "bf16")
        rows = A.KvRows(most, M_keep(np.cumsum([0] + counts)))
        n = A.kv_attention_workspace(cache.desc, rows, qd.blob, A.KvMask())
        ws = A.DeviceBuffer(max(n, 16))
        A.kv_attention(cache.desc, rows, qd.blob, A.KvMask(), 0.125, out.blob, ws.ptr, n)
        A.synchronize()
        check_attention(cache, counts, q, "bf16", out.read())


@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("counts,lengths", [([1, 3], [50, 40]), ([40, 70], [90, 70])])
def test_what_masked_slots_hold_does_not_matter(gpu, fmt, counts, lengths):
    """NaN in every slot that no row sees: behind the length, before the window,
    pages of nobody; and in slots that only later rows see."""
    rng = np.random.default_rng(20)
    window, sinks = 20, 3
    cache = M.Cache(fmt, lengths, 2, 128, 16)
    seen = np.zeros((cache.pages, 16), bool)
    for s, (n, length) in enumerate(zip(counts, lengths)):
        see = np.zeros(length, bool)
        for j in range(n):
            see |= M.visible(length - n + j, length, window, sinks, 1)
        slot = np.nonzero(see)[0]
        seen[cache.table[s, slot // 16], slot % 16] = True
    for name in ("k", "v"):
        if fmt == "4bit":
            x = cache.host[name + "_scale"].transpose(0, 2, 1, 3).copy()
            x[~seen] = 255
            cache.host[name + "_scale"] = np.ascontiguousarray(x.transpose(0, 2, 1, 3))
        else:
            x = cache.host[name].transpose(0, 2, 1, 3).copy()
            x[~seen] = 0x7fc0
            x[~seen, :, ::2] = 0xff80
            cache.host[name] = np.ascontiguousarray(x.transpose(0, 2, 1, 3))
    cache.upload()
    q = new_rows(rng, counts, 4, 128, "bf16")
    got = run_attention(cache, counts, q, "bf16", window, sinks)
    assert np.isfinite(got).all()
    check_attention(cache, counts, q, "bf16", got, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("count", [4, 60, 150])
def test_values_that_only_later_rows_see(gpu, dtype, fmt, count):
    """An infinite or NaN value reaches the rows that see it and no other."""
    rng = np.random.default_rng(21)
    length = 200
    cache = M.Cache(fmt, [length], 2, 64, 16)
    for slot, feature in [(length - 2, 5), (length - count // 2, 40)]:
        page = cache.table[0, slot // 16]
        if fmt == "4bit":
            cache.host["v_scale"][page, 1, slot % 16, feature // 32] = 255
        else:
            cache.host["v"][page, 1, slot % 16, feature] = 0x7f80 if feature == 5 else 0x7fc0
    cache.upload()
    q = new_rows(rng, [count], 4, 64, dtype)
    got = run_attention(cache, [count], q, dtype)
    assert np.isfinite(got[:count - count // 2 - 1]).all() and np.isfinite(got[:, :2]).all()
    assert not np.isfinite(got[-1, 2:]).all()
    check_attention(cache, [count], q, dtype, got)


def test_keys_that_are_not_finite(gpu):
    """A NaN key makes the rows that see it NaN; a row of large scores stays right."""
    rng = np.random.default_rng(22)
    cache = M.Cache("bf16", [100], 1, 64, 16)
    cache.host["k"][cache.table[0, 98 // 16], 0, 98 % 16, 3] = 0x7fc0
    cache.upload()
    q = new_rows(rng, [4], 2, 64, "f32", std=30.0)
    got = run_attention(cache, [4], q, "f32")
    assert np.isfinite(got[:2]).all() and np.isnan(got[2:]).all()
    k, _ = cache.rows("k", 0)
    v, _ = cache.rows("v", 0)
    want, bound = M.attention(q[:2], k[:98], v[:98], 98, 0, 0, 1, 0.125, "f32")
    assert (np.abs(got[:2] - want) <= bound).all()


@pytest.mark.parametrize("count", [3, 70])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales(gpu, count, dtype):
    """Zero (the mean), negative and large scales."""
    rng = np.random.default_rng(23)
    cache = M.Cache("bf16", [77], 2, 64, 16)
    cache.upload()
    q = new_rows(rng, [count], 2, 64, dtype)
    for scale in (0.0, -0.25, 20.0, 1e-30):
        got = run_attention(cache, [count], q, dtype, scale=scale)
        k, _ = cache.rows("k", 0)
        v, _ = cache.rows("v", 0)
        want, bound = M.attention(q, k * np.sign(scale or 1.0), v, 77, 0, 0, 1, abs(scale), dtype)
        assert (np.abs(got - want) <= bound).all(), scale


def test_no_visible_key_gives_zeros(gpu):
    """Every page that a row sees is none of the pool's."""
    rng = np.random.default_rng(24)
    for counts, length in ([1], 900), ([50], 60):
        cache = M.Cache("bf16", [length], 2, 64, 16)
        cache.table[:] = cache.pages
        cache.upload()
        q = new_rows(rng, counts, 2, 64, "bf16")
        got = run_attention(cache, counts, q, "bf16")
        assert (got == 0).all()
        assert cache.status() == A.KV_BAD_PAGE


@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("count", [1, 40, 300])
def test_pages_that_no_row_sees_may_be_given_back(gpu, fmt, count):
    """Table entries between the first slots and the window name no page: they
    are not needed, also where a visible slot is next to theirs."""
    rng = np.random.default_rng(48)
    for length, window, sinks in ((700, 50, 5), (701, 47, 0), (716, 64, 17), (690, 33, 40)):
        cache = M.Cache(fmt, [length], 2, 64, 16)
        seen = np.zeros(length, bool)
        for j in range(count):
            seen |= M.visible(length - count + j, length, window, sinks, 1)
        for page in range(cache.width):
            if not seen[16 * page:16 * page + 16].any():
                cache.table[0, page] = -1
        assert (cache.table < 0).any()
        cache.upload()
        q = new_rows(rng, [count], 4, 64, "bf16")
        got = run_attention(cache, [count], q, "bf16", window, sinks)
        check_attention(cache, [count], q, "bf16", got, window, sinks)
        assert cache.status() == 0


def test_same_bits_every_time_and_on_another_stream(gpu):
    rng = np.random.default_rng(25)
    for counts, lengths in ([1, 1], [3000, 800]), ([200, 3], [900, 1200]):
        cache = M.Cache("4bit", lengths, 2, 128, 16)
        cache.upload()
        q = new_rows(rng, counts, 4, 128, "bf16")
        first = run_attention(cache, counts, q, "bf16")
        check_attention(cache, counts, q, "bf16", first)
        stream = A.Stream()
        for s in (None, stream):
            np.testing.assert_array_equal(run_attention(cache, counts, q, "bf16", stream=s), first)
        stream.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
def test_in_place_and_two_calls_at_once(gpu, fmt, dtype):
    """Queries become the output, on two streams side by side with a workspace each."""
    rng = np.random.default_rng(50)
    calls = []
    for counts, lengths in ([1, 3, 1], [4000, 70, 9]), ([1, 260, 2], [5000, 800, 2]), ([300], [2000]):
        cache = M.Cache(fmt, lengths, 2, 128, 16)
        cache.upload()
        q = new_rows(rng, counts, 6, 128, dtype)
        calls.append((cache, counts, q, run_attention(cache, counts, q, dtype)))
    streams = [A.Stream(), A.Stream()]
    held = []
    for _ in range(3):
        for i, (cache, counts, q, _) in enumerate(calls):
            rows = A.KvRows(max(counts), M_keep(np.cumsum([0] + counts)))
            x = M.Rows(q, dtype)
            n = A.kv_attention_workspace(cache.desc, rows, x.blob, A.KvMask())
            held.append((i, x, A.DeviceBuffer(max(n, 16)), n, rows))
    A.synchronize()
    for j, (i, x, ws, n, rows) in enumerate(held):
        A.kv_attention(calls[i][0].desc, rows, x.blob, A.KvMask(), 128 ** -0.5, x.blob, ws.ptr, n, streams[j % 2])
    for stream in streams:
        stream.synchronize()
    for i, x, *_ in held:
        np.testing.assert_array_equal(x.read(), calls[i][3])
    for cache, counts, q, got in calls:
        check_attention(cache, counts, q, dtype, got)
    for stream in streams:
        stream.destroy()


def test_shared_pages(gpu):
    """Two sequences with the same first pages, and one page named twice."""
    rng = np.random.default_rng(26)
    cache = M.Cache("bf16", [60, 70], 1, 64, 16)
    cache.table[1, :3] = cache.table[0, :3]
    cache.table[0, 2] = cache.table[0, 0]
    cache.upload()
    q = new_rows(rng, [2, 30], 2, 64, "bf16")
    got = run_attention(cache, [2, 30], q, "bf16")
    check_attention(cache, [2, 30], q, "bf16", got)


def test_long_cache_passes_32_bits(gpu):
    """Pools of 4.5 GiB: rows whose byte offsets pass 2^32 and 2^31."""
    pages, page, heads, dim = 9 * 1024, 256, 8, 128
    size = pages * page * heads * dim * 2
    assert size > 1 << 32
    rng = np.random.default_rng(27)
    k_pool, v_pool = A.DeviceBuffer(size), A.DeviceBuffer(size)
    table = np.array([[pages - 1, 4097, 8191, 0]], np.int32)
    td, ld = M.ints(table), M.ints([600])
    desc = A.KvCache(A.KV_BF16, pages, page, heads, dim, k_pool.ptr, v_pool.ptr, td.ptr, 1, 4, ld.ptr)
    k, v = (new_rows(rng, [600], heads, dim, "bf16") for _ in range(2))
    rows = A.KvRows(600)
    A.kv_append(desc, rows, M.Rows(k, "bf16").blob, M.Rows(v, "bf16").blob)
    ko, vo = (M.Rows(np.zeros(k.shape), "bf16") for _ in range(2))
    A.kv_read(desc, rows, ko.blob, vo.blob)
    A.synchronize()
    np.testing.assert_array_equal(ko.read(), k)
    np.testing.assert_array_equal(vo.read(), v)
    q = new_rows(rng, [600], heads, dim, "bf16")
    for n in (2, 600):
        part = M.Rows(q[600 - n:], "bf16")
        out = M.Rows(np.zeros(part.shape), "bf16")
        r = A.KvRows(n)
        nb = A.kv_attention_workspace(desc, r, part.blob, A.KvMask(max_length=600))
        ws = A.DeviceBuffer(max(nb, 16))
        A.kv_attention(desc, r, part.blob, A.KvMask(max_length=600), dim ** -0.5, out.blob, ws.ptr, nb)
        A.synchronize()
        got = out.read()
        want, bound = M.attention(q[598:], k.astype(np.float64), v.astype(np.float64), 600, 0, 0, 1, dim ** -0.5, "bf16")
        assert (np.abs(got[-2:] - want) <= bound).all()


# ---- a session ----

@pytest.mark.parametrize("fmt", ["bf16", "4bit"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_session(gpu, fmt, dtype):
    """Text first, then frames that see each other, then single tokens, for
    two sequences of different lengths: every step's append and attention
    against the 64-bit model of the whole session."""
    rng = np.random.default_rng(30)
    heads, kv_heads, dim, page, sinks, window = 4, 2, 128, 16, 6, 48
    steps = [([6, 6], 1), ([16, 16], 16), ([16, 0], 16), ([16, 16], 16), ([1, 1], 1), ([0, 1], 1), ([3, 1], 1)]
    cache = M.Cache(fmt, [80, 60], kv_heads, dim, page)
    cache.lengths[:] = 0
    desc = cache.upload()
    rope = A.Rope(126, 3)
    for counts, block in steps:
        total = sum(counts)
        q, k, v = (new_rows(rng, [total], h, dim, dtype) for h in (heads, kv_heads, kv_heads))
        pos = rng.integers(0, 100, (total, 3))
        cache.set(lengths=cache.lengths + np.array(counts))
        qd, out = M.Rows(q, dtype), M.Rows(np.zeros(q.shape), dtype)
        rows = A.KvRows(max(counts), M_keep(np.cumsum([0] + counts)))
        mask = A.KvMask(window, sinks, block)
        A.kv_append(desc, rows, M.Rows(k, dtype).blob, M.Rows(v, dtype).blob, rope, M_keep(pos), qd.blob, qd.blob)
        n = A.kv_attention_workspace(desc, rows, qd.blob, mask)
        ws = A.DeviceBuffer(max(n, 16))
        A.kv_attention(desc, rows, qd.blob, mask, dim ** -0.5, out.blob, ws.ptr, n)
        A.synchronize()
        assert cache.status() == 0
        kr = M.rotate(k, pos, 126, 3)
        check_pools(cache, expected_pools(cache, counts, kr, v.astype(np.float64)), counts, k,
                    {"rows": kr, "kw": {"rope_dim": 126, "axes": 3}})
        cache.host = cache.download()
        check_attention(cache, counts, qd.read(), dtype, out.read(), window, sinks, block)


def hip():
    """The HIP runtime that the library is linked with."""
    A.lib()
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64.so" in line)
    return ctypes.CDLL(path)


def test_captured_step_follows_the_lengths(gpu):
    """An append, an attention and a read in a graph, replayed while lengths
    and inputs change, with the same calls made eagerly between the replays."""
    rng = np.random.default_rng(31)
    cache = M.Cache("4bit", [6000, 9000], 2, 128, 16)
    cache.lengths[:] = [400, 900]
    desc = cache.upload()
    shapes = {"q": 4, "k": 2, "v": 2, "qo": 4, "out": 4, "kr": 2, "vr": 2}
    t = {n: M.Rows(np.zeros((2, h, 128)), "bf16") for n, h in shapes.items()}
    rows, mask, rope = A.KvRows(1), A.KvMask(0, 4, 1), A.Rope(128, halves=True)
    n = A.kv_attention_workspace(desc, rows, t["q"].blob, mask)
    assert n > 0
    ws = A.DeviceBuffer(n)
    stream, rt = A.Stream(), hip()

    def step():
        A.kv_append(desc, rows, t["k"].blob, t["v"].blob, rope, None, t["q"].blob, t["qo"].blob, stream)
        A.kv_attention(desc, rows, t["qo"].blob, mask, 128 ** -0.5, t["out"].blob, ws.ptr, n, stream)
        A.kv_read(desc, rows, t["kr"].blob, t["vr"].blob, stream)

    def results():
        stream.synchronize()
        return {m: t[m].read() for m in ("qo", "out", "kr", "vr")}

    step()
    stream.synchronize()
    s, graph, run = ctypes.c_void_p(stream.handle), ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(s, 2) == 0  # relaxed: other calls may go on
    step()
    assert rt.hipStreamEndCapture(s, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for i in range(4):
        for m in ("q", "k", "v"):
            t[m].buf.upload(A.f32_to_bf16_bits(rng.standard_normal(t[m].shape).astype(np.float32)))
        cache.set(lengths=[401 + 1300 * i, 901 + 2600 * i])
        assert rt.hipGraphLaunch(run, s) == 0
        replayed = results()
        pools = cache.download()
        for m in ("qo", "out", "kr", "vr"):
            t[m].buf.zero()
        A.synchronize()
        step()
        for m, x in results().items():
            np.testing.assert_array_equal(replayed[m], x)
        for name, x in cache.download().items():
            np.testing.assert_array_equal(pools[name], x)
        cache.host = pools
        for j in range(2):
            k, _ = cache.rows("k", j)
            v, _ = cache.rows("v", j)
            want, bound = M.attention(replayed["qo"][j:j + 1], k, v, int(cache.lengths[j]), 0, 4, 1, 128 ** -0.5,
                                      "bf16")
            assert (np.abs(replayed["out"][j:j + 1] - want) <= bound).all()
    assert rt.hipGraphExecDestroy(run) == 0 and rt.hipGraphDestroy(graph) == 0
    stream.destroy()


def test_captured_mixed_call_follows_its_rows(gpu):
    """One graph of an attention over many sequences, replayed while which of
    them has the chunk, and how long they are, changes; an eager call of the same
    between the replays."""
    rng = np.random.default_rng(32)
    n, most, heads, dim = 400, 600, 8, 64
    cache = M.Cache("bf16", [most + 100] * n, 4, dim, 32)
    desc = cache.upload()
    total = most + n - 1 + 5  # rows behind the last sequence among them
    q, out = M.Rows(np.zeros((total, heads, dim)), "bf16"), M.Rows(np.zeros((total, heads, dim)), "bf16")
    cu = M.ints(np.zeros(n + 1))
    rows, mask = A.KvRows(most, cu.ptr), A.KvMask(0, 0, 1, most + 100)
    need = A.kv_attention_workspace(desc, rows, q.blob, mask)
    assert need > 0  # the parts' numbers among it
    ws, other = A.DeviceBuffer(max(need, 16)), A.DeviceBuffer(max(need, 16))
    stream, rt = A.Stream(), hip()

    def step(workspace):
        A.kv_attention(desc, rows, q.blob, mask, dim ** -0.5, out.blob, workspace.ptr, need, stream)

    def set_rows(i):
        counts = [1] * n
        counts[(7 + 41 * i) % n] = most - 50 * i
        counts[(20 + 3 * i) % n] = 0
        cu.upload(np.cumsum([0] + counts).astype(np.int32))
        cache.set(lengths=[c + int(x) for c, x in zip(counts, rng.integers(0, 100, n))])
        return counts

    set_rows(0)
    step(ws)
    stream.synchronize()
    s, graph, run = ctypes.c_void_p(stream.handle), ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(s, 2) == 0
    step(ws)
    assert rt.hipStreamEndCapture(s, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for i in range(1, 4):
        counts = set_rows(i)
        x = new_rows(rng, [total], heads, dim, "bf16", std=2.0)
        q.buf.upload(A.f32_to_bf16_bits(x))
        out.buf.upload(A.f32_to_bf16_bits(np.full(x.shape, 5.0, np.float32)))
        A.synchronize()
        assert rt.hipGraphLaunch(run, s) == 0
        stream.synchronize()
        replayed = out.read()
        assert (replayed[sum(counts):] == 5.0).all()
        out.buf.zero()
        A.synchronize()
        step(other)
        stream.synchronize()
        np.testing.assert_array_equal(out.read()[:sum(counts)], replayed[:sum(counts)])
        check_attention(cache, counts, x, "bf16", replayed)
    assert rt.hipGraphExecDestroy(run) == 0 and rt.hipGraphDestroy(graph) == 0
    stream.destroy()
