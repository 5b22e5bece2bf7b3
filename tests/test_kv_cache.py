"""The key/value cache on the host: what a row sees and how the keys are dealt
out, what of a call's device data is taken, and the refusals. No GPU needed."""

import ctypes

import numpy as np
import pytest

import awa_hip as A
import kv_model as M


def span(window, sinks, block, slot, length):
    out = (ctypes.c_int * 3)()
    A.lib().awa_kv_host_span(window, sinks, block, slot, length, out)
    return tuple(out)


@pytest.mark.parametrize("window,sinks,block", [(0, 0, 1), (1, 0, 1), (5, 0, 1), (5, 3, 1), (0, 4, 1), (7, 64, 1),
                                                (0, 0, 4), (8, 3, 4), (3, 2, 4), (1, 9, 4), (6, 5, 5), (40, 1, 7)])
def test_span_is_the_mask(window, sinks, block):
    for length in (1, 2, 7, 30):
        last = (0, 0, 0)
        for slot in range(length):
            s = span(window, sinks, block, slot, length)
            assert 0 <= s[0] <= s[1] <= s[2] <= length
            assert all(a <= b for a, b in zip(last, s))  # all three grow
            last = s
            k = np.arange(length)
            np.testing.assert_array_equal((k < s[0]) | ((k >= s[1]) & (k < s[2])),
                                          M.visible(slot, length, window, sinks, block))


def test_span_at_the_largest_sizes():
    top = 1 << 30
    for window, sinks, block in [(top, top, top), (0, 0, top), (1, top, 1), (top, 0, 1), (top, 1, top - 1)]:
        for slot, length in [(0, 1), (top - 1, top), (0, top), (top // 2, top)]:
            e = sinks + block * -(-(slot + 1 - sinks) // block)
            end = min(e, length)
            begin = min(max(0, e - window) if window else 0, end)
            assert span(window, sinks, block, slot, length) == (min(sinks, begin), begin, end)


@pytest.mark.parametrize("shift", [4, 5, 6])
def test_tiles_hold_every_visible_key_once(shift):
    rng = np.random.default_rng(shift)
    for _ in range(300):
        window, sinks, block = (int(x) for x in (rng.integers(0, 200), rng.integers(0, 150), rng.choice([1, 1, 16, 33])))
        length = int(rng.integers(1, 700))
        a = int(rng.integers(0, length))
        b = int(rng.integers(a, length))
        first, last = span(window, sinks, block, a, length), span(window, sinks, block, b, length)
        out = (ctypes.c_int * 3)()
        A.lib().awa_kv_host_tiles((ctypes.c_int * 3)(*first), (ctypes.c_int * 3)(*last), shift, out)
        n_sinks, begin, rest = out
        tiles = list(range(n_sinks)) + list(range(begin, begin + rest))
        assert len(set(tiles)) == len(tiles)
        seen = np.zeros(length, bool)
        for slot in range(a, b + 1):
            seen |= M.visible(slot, length, window, sinks, block)
        need = set((np.nonzero(seen)[0] >> shift).tolist())
        assert need <= set(tiles)
        assert all(t << shift < length for t in tiles)  # no tile without a slot of the sequence


@pytest.mark.parametrize("first,end,length,bad", [
    (0, 3, 3, 0), (0, 0, 0, 0), (2, 2, 5, 0), (4, 8, 64, 0), (-1, 2, 5, A.KV_BAD_ROWS), (3, 2, 5, A.KV_BAD_ROWS),
    (6, 11, 20, A.KV_BAD_ROWS), (0, 6, 20, A.KV_BAD_ROWS), (0, 3, -1, A.KV_BAD_LENGTH), (0, 3, 65, A.KV_BAD_LENGTH),
    (0, 3, 2, A.KV_BAD_LENGTH), (0, 6, 65, A.KV_BAD_LENGTH | A.KV_BAD_ROWS),
    (-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1, A.KV_BAD_LENGTH | A.KV_BAD_ROWS)])
def test_sequences_that_do_not_fit_have_no_rows(first, end, length, bad):
    out = (ctypes.c_int * 4)()
    A.lib().awa_kv_host_sequence(first, end, length, 64, 5, 10, out)
    assert out[3] == bad
    assert out[1] == (0 if bad else end - first)


def cache(**kw):
    d = dict(fmt=A.KV_BF16, pages=4, page_tokens=16, kv_heads=2, head_dim=128, k=4096, v=4096, page_table=4096,
             sequences=1, table_width=4, lengths=4096)
    d.update(kw)
    return A.KvCache(**d)


def rows(heads=2, total=3, size=2, dim=128, ptr=4096, **kw):
    return A.mat(ptr, dim, heads, total, size, dims=3, **kw)


BAD_CACHES = [dict(fmt=2), dict(fmt=-1), dict(pages=0), dict(pages=-4), dict(pages=1 << 27, page_tokens=16, kv_heads=1), dict(page_tokens=8), dict(page_tokens=24),
              dict(page_tokens=2048), dict(page_tokens=0), dict(kv_heads=0), dict(kv_heads=70000), dict(head_dim=96),
              dict(head_dim=256), dict(sequences=0), dict(sequences=65536), dict(table_width=0),
              dict(table_width=1 << 27), dict(table_width=4, table_stride=3), dict(k=0), dict(v=0), dict(k=4104),
              dict(v=4097), dict(page_table=0), dict(page_table=4098), dict(lengths=0), dict(lengths=4097),
              dict(status=4099), dict(fmt=A.KV_MXFP4), dict(fmt=A.KV_MXFP4, k_scale=4096),
              dict(fmt=A.KV_MXFP4, k_scale=4096, v_scale=4097)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(kw):
    c, r = cache(**kw), A.KvRows(3, 4096)
    dim = c.head_dim
    heads = max(1, min(c.kv_heads, 4))
    b = rows(heads=heads, dim=dim)
    for call in (lambda: A.kv_append(c, r, b, b), lambda: A.kv_read(c, r, b, b),
                 lambda: A.kv_attention_workspace(c, r, b, A.KvMask()),
                 lambda: A.kv_attention(c, r, b, A.KvMask(), 1.0, b, 4096, 1 << 40)):
        with pytest.raises(A.AwaError) as e:
            call()
        assert e.value.code == A.AWA_ERR_INVALID


@pytest.mark.parametrize("make", [
    lambda: (A.KvRows(0, 4096), rows()), lambda: (A.KvRows(-1, 4096), rows()), lambda: (A.KvRows(2 ** 31 - 1, 4096), rows()),
    lambda: (A.KvRows(2), rows()),            # 1 sequence of 2 rows, 3 rows in the blobs
    lambda: (A.KvRows(3, 4097), rows()),
    lambda: (A.KvRows(3, 4096), rows(ptr=0)), lambda: (A.KvRows(3, 4096), rows(ptr=4104)),
    lambda: (A.KvRows(3, 4096), rows(size=2, cstep=260)),   # rows off 16-byte addresses
    lambda: (A.KvRows(3, 4096), rows(cstep=128)),           # rows overlap
    lambda: (A.KvRows(3, 4096), rows(dim=64)), lambda: (A.KvRows(3, 4096), rows(total=0)),
    lambda: (A.KvRows(3, 4096), rows(size=1)),
    lambda: (A.KvRows(3, 4096), A.mat(4096, 128, 2, 3, 2, dims=2)),
    lambda: (A.KvRows(3, 4096), A.mat(4096, 128, 2, 3, 2, dims=3, n=2))])
def test_bad_rows_are_refused_by_every_call(make):
    r, b = make()
    c = cache()
    for call in (lambda: A.kv_append(c, r, b, b), lambda: A.kv_read(c, r, b, b),
                 lambda: A.kv_attention_workspace(c, r, b, A.KvMask()),
                 lambda: A.kv_attention(c, r, b, A.KvMask(), 1.0, b, 4096, 1 << 40)):
        with pytest.raises(A.AwaError) as e:
            call()
        assert e.value.code == A.AWA_ERR_INVALID


def refused(call):
    with pytest.raises(A.AwaError) as e:
        call()
    assert e.value.code == A.AWA_ERR_INVALID


def test_append_refusals():
    c, r, b = cache(), A.KvRows(3, 4096), rows()
    rope, axes3 = A.Rope(128), A.Rope(126, 3)
    refused(lambda: A.kv_append(c, r, b, rows(heads=3)))
    refused(lambda: A.kv_append(c, r, b, rows(total=4)))
    refused(lambda: A.kv_append(c, r, b, rows(size=4)))          # two types
    refused(lambda: A.kv_append(c, r, b, b, rope, None, rows(4)))  # q without q_out
    refused(lambda: A.kv_append(c, r, b, b, rope, None, None, rows(4)))
    refused(lambda: A.kv_append(c, r, b, b, None, None, rows(4), rows(4)))  # q without a rope
    refused(lambda: A.kv_append(c, r, b, b, rope, None, rows(4), rows(5)))
    refused(lambda: A.kv_append(c, r, b, b, rope, None, rows(4, size=4), rows(4, size=4)))
    refused(lambda: A.kv_append(c, r, b, b, rope, None, rows(4), rows(4, size=4)))
    refused(lambda: A.kv_append(c, r, b, b, rope, None, rows(4, total=2), rows(4, total=2)))
    refused(lambda: A.kv_append(c, r, b, b, axes3))              # axes without positions
    refused(lambda: A.kv_append(c, r, b, b, rope, 4098))
    small = rows(dim=64)
    refused(lambda: A.kv_append(cache(head_dim=64), r, small, small, rope))  # rope beyond the head
    refused(lambda: A.kv_read(c, r, b, rows(size=4)))
    refused(lambda: A.kv_read(c, r, b, rows(heads=4)))


def test_attention_refusals():
    c, r = cache(), A.KvRows(3, 4096)
    q = rows(heads=4)
    ok = A.KvMask(8, 2, 1)
    for mask in (A.KvMask(-1), A.KvMask(0, -1), A.KvMask(0, 0, 0), A.KvMask(0, 0, 1, -1), A.KvMask((1 << 30) + 1),
                 A.KvMask(0, 2 ** 31 - 1), A.KvMask(0, 0, 2 ** 31 - 1)):
        refused(lambda: A.kv_attention(c, r, q, mask, 1.0, q, 4096, 1 << 40))
        refused(lambda: A.kv_attention_workspace(c, r, q, mask))
    refused(lambda: A.kv_attention(c, r, rows(heads=3), ok, 1.0, rows(heads=3), 4096, 1 << 40))
    for scale in (float("nan"), float("inf")):
        refused(lambda: A.kv_attention(c, r, q, ok, scale, q, 4096, 1 << 40))
    refused(lambda: A.kv_attention(c, r, q, ok, 1.0, rows(heads=2), 4096, 1 << 40))
    refused(lambda: A.kv_attention(c, r, q, ok, 1.0, rows(heads=4, size=4), 4096, 1 << 40))
    refused(lambda: A.kv_attention(c, r, q, ok, 1.0, rows(heads=4, total=2), 4096, 1 << 40))


def test_workspace_is_asked_for():
    """A call whose keys are dealt to several workgroups needs its bytes, 16-byte aligned."""
    c, r, q = cache(table_width=1024), A.KvRows(1), rows(heads=2, total=1)
    n = A.kv_attention_workspace(c, r, q, A.KvMask())
    assert n > 0 and n % 4 == 0
    refused(lambda: A.kv_attention(c, r, q, A.KvMask(), 1.0, q))
    refused(lambda: A.kv_attention(c, r, q, A.KvMask(), 1.0, q, 4096, n - 1))
    refused(lambda: A.kv_attention(c, r, q, A.KvMask(), 1.0, q, 4100, n))
    # One short sequence is one workgroup a head.
    assert A.kv_attention_workspace(c, r, q, A.KvMask(max_length=64)) == 0


def test_workspace_of_single_tokens_beside_chunks():
    """Parts are kept of a call's rows alone, however many sequences it has, and
    of sequences of one row tile alone where longer ones fill the device."""
    def bytes_of(sequences, total, most, max_length, heads=8, kv_heads=2):
        c = cache(kv_heads=kv_heads, sequences=sequences, table_width=8192)
        return A.kv_attention_workspace(c, A.KvRows(most, 4096), rows(heads=heads, total=total), A.KvMask(max_length=max_length))

    part = 8 * 130 * 4  # a row of a part, of all heads, bytes
    # Chunks of many row tiles, which are not split: none can have few rows.
    assert bytes_of(60, 60 * 500, 500, 60000) == 0
    for sequences, total, most in ((2, 4097, 4096), (60, 5000, 4096), (60, 700, 300), (1000, 5095, 4096)):
        n = bytes_of(sequences, total, most, 60000)
        numbers = -(-2 * (sequences + 1) * 4 // 16) * 16  # of the parts' list
        assert n > 0 and (n % part == 0 or (n - numbers) % part == 0)
        assert n <= 2 * 64 * part * total + numbers
    # Of 1000 sequences at most 32 rows of each are in one row tile.
    assert bytes_of(1000, 10 ** 6, 9 * 10 ** 5, 60000) <= 64 * part * 32000 + 10 ** 4


def test_calls_of_too_many_workgroups_are_refused():
    def ask(sequences, total, most, kv_heads, heads, max_length=0):
        c = cache(kv_heads=kv_heads, sequences=sequences, table_width=1024)
        return A.kv_attention_workspace(c, A.KvRows(most, 4096), rows(heads=heads, total=total), A.KvMask(max_length=max_length))

    assert ask(65535, 65535, 1, 20, 20, 64) == 0
    # Many short sequences beside a long one: numbered through, not all as long.
    for sequences, most, heads in ((4000, 16384, 32), (65535, 4096, 24)):
        assert ask(sequences, most + sequences - 1, most, 8, heads, 64) < 10 ** 6
    for args in ((65535, 65535, 1, 65535, 65535), (65535, 1 << 25, 500, 300, 300), (1, 1 << 24, 1 << 24, 8, 64),
                 (1, 1 << 22, 1 << 22, 300, 300), (2, 2, 1, 1, 1 << 30)):
        refused(lambda: ask(*args))
    big = rows(total=(1 << 25) + 1)
    refused(lambda: A.kv_append(cache(), A.KvRows(5, 4096), big, big))
    refused(lambda: A.kv_read(cache(), A.KvRows(5, 4096), big, big))


@pytest.mark.parametrize("args", [(0,), (130,), (7,), (128, 5), (-2,), (64, 0), (12, 3, -1.0), (128, 1, 0.0),
                                  (128, 1, float("nan")), (128, 1, float("inf")), (126, 3, 1e4, True), (24, 1, 1e4, True)])
def test_rope_refusals(args):
    refused(lambda: A.Rope(*args))


def test_rope_frequencies_are_checked():
    with pytest.raises(ValueError):
        A.Rope(16, frequencies=[1.0] * 7)
    refused(lambda: A.Rope(16, frequencies=[1.0] * 7 + [float("nan")]))
    refused(lambda: A.Rope(16, frequencies=[1.0] * 7 + [float("inf")]))
    A.Rope(16, frequencies=[1.0] * 8).destroy()


def test_model_of_the_four_bit_rows():
    """The oracle's codes: every value that e2m1 holds comes back, ties go to
    the even code, and no value is off by more than half its step."""
    grid = np.concatenate([M.GRID, -M.GRID] * 2)
    codes, byte = M.encode4(grid)
    assert byte == 127
    np.testing.assert_array_equal(M.decode4(codes, byte), grid)
    x = np.zeros(32)
    x[:8] = [7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    codes, byte = M.encode4(x)
    np.testing.assert_array_equal(M.decode4(codes, byte)[:8], [6, 0, 1, 1, 2, 2, 4, 4])
    assert M.encode4(x * (1 + 2.0 ** -40))[1] == 128
    rng = np.random.default_rng(0)
    x = rng.standard_normal((100, 64)) * np.exp2(rng.integers(-30, 30, (100, 1)))
    codes, byte = M.encode4(x)
    unit = np.repeat(np.ldexp(1.0, byte.astype(int) - 127), 32, -1)
    y = np.abs(x) / unit
    step = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))
    assert (np.abs(M.decode4(codes, byte) - x) <= step / 2 * unit).all()


def test_division_by_a_multiplication():
    """Every divisor to 200 and large ones, at multiples and beside them, up to 2^30."""
    rng = np.random.default_rng(1)
    divide = A.lib().awa_kv_host_divide
    for d in list(range(1, 201)) + [1 << 10, (1 << 10) + 1, 65535, 65536, 65537, (1 << 29) + 3, (1 << 30) - 1]:
        top = (1 << 30) - 1
        q = [0, 1, top // d] + [int(x) for x in rng.integers(0, top // d + 1, 30)]
        for n in {x for k in q for x in (k * d - 1, k * d, k * d + 1, k * d + d - 1)} | {top, 0}:
            if 0 <= n <= top:
                assert divide(n, d) == n // d, (n, d)
