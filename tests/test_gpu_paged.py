"""The paged key/value cache on the GPU against its restatement in NumPy's 64-bit integers: every result is equal, bit for bit."""
import numpy as np
import pytest

from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


def tables(rows, hd, fa):
    from integer_inference_engine_b200.model import rope_tables
    return tuple(np.ascontiguousarray(t, np.int64) for t in rope_tables(max(1, rows), hd, 50000.0, fa))


def pool(rng, lengths, P, Hkv, hd, bits, spare=3):
    """Pages in random order, a table whose unused entries point nowhere, rows of garbage behind every sequence's last."""
    per = max(1, max((n + P - 1) // P for n in lengths)) + 1
    need = sum((n + P - 1) // P for n in lengths)
    order, at = rng.permutation(need + spare).astype(np.int32), 0
    table = np.full((len(lengths), per), -7, np.int32)
    for b, n in enumerate(lengths):
        m = (n + P - 1) // P
        table[b, :m] = order[at:at + m]
        at += m
    draw = lambda: rng.integers(-(1 << bits), 1 << bits, size=(need + spare, Hkv, P, hd), dtype=np.int64).astype(np.int32)
    return draw(), draw(), table


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def attend(q, kp, vp, table, lengths, **kw):
    from integer_inference_engine_b200 import device
    kw = {k: dev(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    return device.paged_attention(q if hasattr(q, "is_cuda") else dev(q), dev(kp), dev(vp), dev(table), dev(np.array(lengths, np.int32)), **kw).cpu().numpy()


# heads, KV heads, head dimension, page rows, lengths, window, rope, fa, bits of q, bits of keys and values
ATTEND = [
    (8, 2, 64, 16, [0, 1, 15, 16, 17, 127], 0, 1, 16, 18, 18),
    (8, 1, 128, 16, [128, 129, 255, 257, 0, 300], 0, 2, 16, 18, 18),
    (4, 4, 128, 32, [1, 33, 700], 0, 0, 16, 18, 30),
    (16, 2, 128, 64, [1000, 64, 65], 0, 1, 16, 19, 19),
    (12, 4, 64, 8, [9, 200], 0, 2, 16, 20, 31),
    (6, 2, 96, 16, [130, 5], 0, 1, 16, 18, 18),
    (5, 5, 32, 24, [100, 23, 24, 25], 0, 1, 16, 18, 18),
    (12, 1, 128, 16, [150, 40], 0, 1, 16, 18, 18),
    (20, 1, 64, 16, [150, 1], 0, 2, 16, 18, 18),
    (4, 2, 128, 128, [129, 1, 500], 0, 1, 16, 18, 18),
    (8, 2, 128, 16, [200, 30, 65, 66], 65, 1, 16, 18, 18),
    (8, 2, 128, 16, [500, 1, 2], 1, 1, 16, 18, 18),
    (8, 2, 64, 32, [500, 129, 128], 128, 2, 16, 18, 18),
    (8, 2, 128, 16, [300, 77], 0, 1, 12, 14, 16),
    (8, 2, 128, 16, [300, 77], 0, 1, 22, 20, 20),
    (8, 2, 64, 16, [200, 3], 0, 1, 25, 20, 20),
    (8, 2, 128, 16, [200, 20], 0, 1, 16, 40, 24),
    (8, 2, 64, 16, [140, 20], 0, 2, 16, 61, 31),
    (4, 2, 128, 16, [150], 0, 0, 16, 63, 31),
    (8, 2, 80, 16, [140, 3], 0, 1, 16, 18, 18),
    (4, 2, 256, 16, [140, 3], 0, 2, 16, 18, 18),
    (8, 2, 128, 5, [140, 3, 5, 6], 0, 1, 16, 18, 18),
    (4, 2, 64, 1, [40, 3], 0, 1, 16, 18, 18),
    (4, 1, 2, 16, [40, 3], 0, 1, 16, 18, 18),
    (32, 4, 128, 16, [1500, 3], 0, 1, 16, 18, 18),
    (8, 8, 128, 16, list(range(0, 60, 1)), 0, 1, 16, 18, 18),
]


@pytest.mark.parametrize("shape", ATTEND, ids=[f"{i}-{c[0]}x{c[1]}x{c[2]}-p{c[3]}" for i, c in enumerate(ATTEND)])
def test_attention(shape):
    from integer_inference_engine_b200 import device
    H, Hkv, hd, P, lengths, window, rope, fa, qbits, kvbits = shape
    rng = np.random.default_rng(hd * 7 + P + len(lengths))
    kp, vp, table = pool(rng, lengths, P, Hkv, hd, kvbits)
    q = rng.integers(-(1 << qbits), 1 << qbits, size=(len(lengths), H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, fa)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, fa=fa, window=window, cos=cos, sin=sin, rope=rope)
    assert device.read_flags() == 0
    want = po.attention(q, kp, vp, table, lengths, fa, window, cos, sin, rope)
    assert np.array_equal(got, want)


@pytest.mark.parametrize(("B", "most", "H", "Hkv", "hd", "P", "window", "seed"), [
    (40, 4500, 4, 4, 64, 16, 0, 1), (12, 9000, 8, 4, 32, 8, 0, 2), (300, 300, 8, 8, 32, 16, 0, 3), (3, 40000, 4, 2, 64, 64, 0, 4), (1, 70000, 2, 1, 32, 128, 0, 5),
    (60, 6000, 8, 2, 128, 32, 1500, 6), (700, 150, 2, 2, 64, 8, 0, 7), (25, 3000, 12, 4, 96, 16, 0, 8)])
def test_long_lists(B, most, H, Hkv, hd, P, window, seed):
    """Enough tiles that every CTA has many: pairs within a CTA, cut between two and more, sequences without keys among them."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(seed)
    lengths = [most] + [int(n) for n in rng.integers(1, most + 1, size=B - 1)]
    if B > 4:
        lengths[B // 2] = lengths[1] = 0
    kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
    q = rng.integers(-(1 << 17), 1 << 17, size=(B, H * hd), dtype=np.int64)
    cos, sin = tables(most, hd, 16)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, window=window, cos=cos, sin=sin, rope=1)
    assert device.read_flags() == 0
    assert np.array_equal(got, po.attention(q, kp, vp, table, lengths, 16, window, cos, sin, 1))


@pytest.mark.parametrize(("P", "hd", "H", "Hkv", "window"), [(16, 128, 8, 2, 0), (16, 64, 4, 4, 0), (32, 128, 8, 1, 100), (8, 128, 6, 2, 0), (64, 64, 12, 2, 300), (5, 64, 4, 2, 0), (128, 128, 8, 2, 0)])
def test_attention_over_chosen_pages(P, hd, H, Hkv, window):
    """Lists with empty entries in front, between and behind, of a page twice, of pages beyond the keys and out of the window, of nothing."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(P + hd)
    lengths = [700, 0, 3 * P, 2 * P + 1, 1]
    kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
    n_sel, per = 7, table.shape[1]
    pages = np.full((len(lengths), Hkv, n_sel), -1, np.int32)
    for b, n in enumerate(lengths):
        m = (n + P - 1) // P
        for g in range(Hkv):
            take = rng.permutation(m)[:n_sel]
            pages[b, g, rng.permutation(n_sel)[:len(take)]] = take
    pages[0, 0, :3] = 2
    pages[3, 0] = -1
    pages[2, Hkv - 1, 0] = 3                                            # the page behind the last: its table entry points nowhere, but no row counts
    table[2, 3] = 0
    q = rng.integers(-(1 << 18), 1 << 18, size=(len(lengths), H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, window=window, cos=cos, sin=sin, rope=1, pages=pages)
    assert device.read_flags() == 0 and per > 3
    assert np.array_equal(got, po.attention(q, kp, vp, table, lengths, 16, window, cos, sin, 1, pages))


@pytest.mark.parametrize("shift", [0, 20, 31])
def test_scores_far_apart(shift):
    """Scores whose distance leaves 32 bits, the largest in one key of a later tile; and all equal ones."""
    H, Hkv, hd, P, n = 8, 1, 128, 16, 520
    rng = np.random.default_rng(shift)
    kp, vp, table = pool(rng, [n], P, Hkv, hd, 30)
    q = np.zeros((1, H * hd), np.int64)
    q[0, ::hd] = rng.integers(1, 9, size=H) << shift
    for t in range(n):
        kp[table[0, t // P], 0, t % P, 0] = -(1 << 30) if t != 300 else (1 << 30) + 12345
    inv = 1 << 16
    got = attend(q, kp, vp, table, [n], inv_sqrt=inv)
    assert np.array_equal(got, po.attention(q, kp, vp, table, [n], 16, 0, None, None, 0, inv_sqrt=inv))
    q[:] = 0
    got = attend(q, kp, vp, table, [n], inv_sqrt=inv)
    assert np.array_equal(got, po.attention(q, kp, vp, table, [n], 16, 0, None, None, 0, inv_sqrt=inv))


def test_extreme_values():
    """The ends of int32 in keys and values, the ends of int64 in queries."""
    H, Hkv, hd, P, n = 8, 2, 64, 16, 150
    rng = np.random.default_rng(2)
    kp, vp, table = pool(rng, [n], P, Hkv, hd, 18)
    ends = np.array([-(1 << 31), (1 << 31) - 1, 0, -1, 1, 0x7F7F7F7F, 0x7F7F7F80, -0x80808080 + (1 << 31)], np.int64)
    kp[:] = rng.choice(ends, size=kp.shape)
    vp[:] = rng.choice(ends, size=vp.shape)
    q = rng.choice(np.array([-(1 << 63), (1 << 63) - 1, 0, -1, 1, 0x7F7F7F7F7F7F7F80, 0x80808080, -0x80808081], np.int64), size=(1, H * hd))
    assert np.array_equal(attend(q, kp, vp, table, [n]), po.attention(q, kp, vp, table, [n], 16, 0, None, None, 0))
    q = rng.integers(-3, 4, size=(1, H * hd), dtype=np.int64)
    assert np.array_equal(attend(q, kp, vp, table, [n]), po.attention(q, kp, vp, table, [n], 16, 0, None, None, 0))


APPEND = [
    # KV heads, head dimension, page rows, rope, positions of the first new rows (negative: none), new rows (None: one each), int32 rows
    (4, 128, 16, 1, [0, 15, 16, -1, 17, 200], None, False),
    (8, 128, 16, 2, [5, 0, 31], [40, 0, 1], False),
    (2, 64, 32, 1, [31, 64, 3], [1, 100, 29], False),
    (1, 256, 8, 0, [7, 0], [9, 8], True),
    (3, 96, 5, 1, [4, 10, 0], [7, 5, 1], False),
    (2, 2, 1, 1, [4, 0], [3, 1], False),
    (2, 80, 64, 2, [-5, 100], [3, 300], False),
    (5, 514, 4, 2, [2], [6], False),
    (2, 128, 128, 1, [100, 127, 0, -1], [200, 2, 128, 4], False),
]


@pytest.mark.parametrize("shape", APPEND, ids=[f"{c[0]}x{c[1]}-p{c[2]}" for c in APPEND])
@pytest.mark.parametrize("bounded", [True, False])
def test_append(shape, bounded):
    import torch

    from integer_inference_engine_b200 import device
    Hkv, hd, P, rope, start, counts, narrow = shape
    rng = np.random.default_rng(hd + P)
    each = counts or [1] * len(start)
    ends = [at + n if at >= 0 else 0 for at, n in zip(start, each)]
    kp, vp, table = pool(rng, ends, P, Hkv, hd, 18)
    bounds = rng.integers(-9, 9, size=(kp.shape[0], Hkv, 2, hd)).astype(np.int32)
    total = sum(each) + 3                                               # rows behind the last sequence's
    kv = rng.integers(-(1 << 18), 1 << 18, size=(total, 3 * Hkv * hd), dtype=np.int64)
    k, v = kv[:, Hkv * hd:2 * Hkv * hd], kv[:, 2 * Hkv * hd:]
    rows = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    cos, sin = tables(max(ends), hd, 16)
    dkv = dev(kv, torch.int32 if narrow else torch.int64)
    dk, dv, dkp, dvp, db = dkv[:, Hkv * hd:2 * Hkv * hd], dkv[:, 2 * Hkv * hd:], dev(kp), dev(vp), dev(bounds)
    device.read_flags()
    for _ in range(2):                                                  # again: the same rows at the same places
        device.paged_append(dk, dv, dkp, dvp, dev(table), dev(np.array(start, np.int32)), rows=None if rows is None else dev(rows), cos=dev(cos), sin=dev(sin), rope=rope,
                            bounds=db if bounded else None)
    assert device.read_flags() == 0
    want_b = bounds.copy()
    po.append(k, v, kp, vp, want_b, table, start, rows, 16, cos, sin, rope)
    assert np.array_equal(dkp.cpu().numpy(), kp) and np.array_equal(dvp.cpu().numpy(), vp)
    assert np.array_equal(db.cpu().numpy(), want_b if bounded else bounds)


def test_append_of_many_sequences():
    """More sequences than a scan takes at once, some without rows."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(8)
    B, Hkv, hd, P = 700, 1, 32, 4
    counts = rng.integers(0, 6, size=B)
    start = rng.integers(-2, 9, size=B)
    ends = [int(a + n) if a >= 0 else 0 for a, n in zip(start, counts)]
    kp, vp, table = pool(rng, ends, P, Hkv, hd, 18)
    bounds = np.zeros((kp.shape[0], Hkv, 2, hd), np.int32)
    rows = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    k, v = (rng.integers(-(1 << 18), 1 << 18, size=(int(rows[-1]), Hkv * hd), dtype=np.int64) for _ in range(2))
    cos, sin = tables(max(ends), hd, 16)
    dkp, dvp, db = dev(kp), dev(vp), dev(bounds)
    device.read_flags()
    device.paged_append(dev(k), dev(v), dkp, dvp, dev(table), dev(start.astype(np.int32)), rows=dev(rows), cos=dev(cos), sin=dev(sin), rope=1, bounds=db)
    assert device.read_flags() == 0
    po.append(k, v, kp, vp, bounds, table, start, rows, 16, cos, sin, 1)
    assert np.array_equal(dkp.cpu().numpy(), kp) and np.array_equal(dvp.cpu().numpy(), vp) and np.array_equal(db.cpu().numpy(), bounds)


def test_bounds_after_going_back():
    """Rows given up and written anew leave nothing behind in the bounds."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(9)
    Hkv, hd, P = 2, 64, 16
    kp, vp, table = pool(rng, [40], P, Hkv, hd, 10)
    db, dkp, dvp = dev(np.zeros((kp.shape[0], Hkv, 2, hd), np.int32)), dev(kp), dev(vp)
    bounds = np.zeros((kp.shape[0], Hkv, 2, hd), np.int32)
    for at, n, bits in ((0, 30, 10), (30, 5, 25), (31, 2, 4)):
        k, v = (rng.integers(-(1 << bits), 1 << bits, size=(n, Hkv * hd), dtype=np.int64) for _ in range(2))
        rows = np.array([0, n], np.int32)
        device.paged_append(dev(k), dev(v), dkp, dvp, dev(table), dev(np.array([at], np.int32)), rows=dev(rows), bounds=db)
        po.append(k, v, kp, vp, bounds, table, [at], rows, 16, None, None, 0)
        assert np.array_equal(db.cpu().numpy(), bounds)


SELECT = [
    # heads, KV heads, head dimension, page rows, lengths, window, rope, pages taken, first, last kept, bits of q
    (8, 2, 128, 16, [1000, 0, 16, 17, 33, 200], 0, 1, 5, 1, 1, 18),
    (8, 8, 64, 32, [700, 1, 95], 0, 2, 3, 1, 2, 18),
    (12, 2, 128, 16, [500, 300], 130, 1, 4, 0, 0, 18),
    (5, 1, 96, 8, [900, 10], 0, 0, 20, 2, 3, 30),
    (16, 1, 64, 5, [400], 0, 1, 7, 1, 1, 50),
    (4, 2, 80, 16, [300], 0, 1, 30, 1, 1, 18),
    (2, 2, 32, 1, [2500, 40], 0, 1, 64, 1, 1, 18),
    (4, 1, 256, 64, [3000], 1000, 1, 6, 0, 1, 18),
    (4, 2, 128, 16, [3000, 1], 0, 1, 1, 0, 1, 18),
    (12, 1, 128, 16, [4000, 2500, 100], 0, 2, 40, 3, 2, 18),
    (8, 8, 128, 8, [20000, 5, 9000], 0, 1, 128, 1, 1, 18),
    (8, 1, 64, 4, [3000], 0, 1, 20, 1, 1, 62),
]


@pytest.mark.parametrize("shape", SELECT, ids=[f"{c[0]}x{c[1]}x{c[2]}-p{c[3]}" for c in SELECT])
@pytest.mark.parametrize("flat", [False, True])
def test_select(shape, flat):
    """flat: bounds of few different values, so that many pages share a score."""
    from integer_inference_engine_b200 import device
    H, Hkv, hd, P, lengths, window, rope, n_select, first, last, qbits = shape
    rng = np.random.default_rng(hd + n_select)
    _, _, table = pool(rng, lengths, P, 1, 2, 4)
    n_pages = table.max() + 1
    bounds = np.sort(rng.integers(-(1 << 18), 1 << 18, size=(n_pages, Hkv, 2, hd)), axis=2)[:, :, ::-1].astype(np.int32)
    if flat:
        bounds[:] = bounds[rng.integers(0, 3, size=n_pages)]
    q = rng.integers(-(1 << qbits), 1 << qbits, size=(len(lengths), H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    device.read_flags()
    got = device.paged_select(dev(q), dev(bounds), dev(table), dev(np.array(lengths, np.int32)), P, n_select, first, last, window=window, cos=dev(cos), sin=dev(sin), rope=rope)
    assert device.read_flags() == 0
    assert np.array_equal(got.cpu().numpy(), po.select(q, bounds, table, lengths, P, n_select, first, last, 16, window, cos, sin, rope))


def test_select_of_many_pages():
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(4)
    hd, n = 32, 9001
    bounds = rng.integers(-40, 40, size=(n, 1, 2, hd)).astype(np.int32)
    table = rng.permutation(n).astype(np.int32)[None]
    q = rng.integers(-3, 4, size=(1, hd), dtype=np.int64)
    for n_select in (2, 1000, 9000, 9001, 9500):
        got = device.paged_select(dev(q), dev(bounds), dev(table), dev(np.array([n], np.int32)), 1, n_select)
        assert np.array_equal(got.cpu().numpy(), po.select(q, bounds, table, [n], 1, n_select, 1, 1, 16, 0, None, None, 0))


# lists of more than 1024 pages, and many of more than 128, ranked by all SMs together
LONG = [
    (12, 1, 128, 16, [20000, 16000, 1], 0, 2, 40, 3, 2, 18),
    (4, 2, 64, 8, [12000, 0, 300, 9000], 5000, 2, 33, 1, 1, 62),
    (8, 4, 80, 4, [5000, 4097, 130], 0, 1, 32, 0, 0, 18),
    (2, 1, 32, 1, [1500, 0, 3, 40, 200] * 9, 0, 1, 30, 1, 1, 18),
    (16, 8, 32, 1, [1100], 0, 0, 1100, 1, 1, 18),
    (3, 1, 16, 2, [2600, 2500], 0, 1, 1, 0, 1, 18),
    (8, 4, 32, 1, [150, 7, 130, 0, 21] * 10, 0, 1, 20, 1, 1, 18),
    (2, 1, 16, 1, [0] * 70 + [140, 129, 12] * 110, 0, 0, 11, 1, 1, 18),
]


@pytest.mark.parametrize("shape", LONG, ids=[f"{c[0]}x{c[1]}x{c[2]}-p{c[3]}" for c in LONG])
@pytest.mark.parametrize("flat", [False, True])
def test_select_from_long_lists(shape, flat):
    test_select(shape, flat)


def test_select_from_a_long_list_with_a_page_outside():
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(12)
    n, hd = 1500, 64
    bounds = np.sort(rng.integers(-1000, 1000, size=(n, 2, 2, hd)), axis=2)[:, :, ::-1].astype(np.int32)
    table = rng.permutation(n).astype(np.int32)[None].repeat(2, 0)
    q = rng.integers(-1000, 1000, size=(2, 4 * hd), dtype=np.int64)
    device.read_flags()
    call = lambda t, lens: device.paged_select(dev(q), dev(bounds), dev(t), dev(np.array(lens, np.int32)), 1, 20, 0, 0).cpu().numpy()
    good = call(table, [n, n - 7])
    assert device.read_flags() == 0
    best = good[0, 0, 0]
    for wrong in (-1, n, 1 << 30):
        other = table.copy()
        other[0, best] = wrong                     # never chosen: the twenty best are others
        got = call(other, [n, n - 7])
        assert device.read_flags() == 16 and best not in got[0] and np.array_equal(got[1], good[1])
    got = call(table, [n + 1, n - 7])              # a length beyond the table: none of its pages
    assert device.read_flags() == 16 and (got[0] == -1).all() and np.array_equal(got[1], good[1])


def test_rows_of_a_wider_matrix_and_a_given_output():
    import torch

    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(6)
    H, Hkv, hd, P, lengths = 8, 2, 128, 16, [90, 7]
    kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
    wide = rng.integers(-(1 << 18), 1 << 18, size=(2, 3 * H * hd), dtype=np.int64)
    q = dev(wide)[:, H * hd:2 * H * hd]
    out = torch.full((2, H * hd), 7, dtype=torch.int64, device="cuda")
    got = device.paged_attention(q, dev(kp), dev(vp), dev(table), dev(np.array(lengths, np.int32)), out=out, max_length=90)
    assert got is out
    assert np.array_equal(out.cpu().numpy(), po.attention(wide[:, H * hd:2 * H * hd], kp, vp, table, lengths, 16, 0, None, None, 0))


def test_what_lies_outside_the_cache_is_flagged_and_left_out():
    import torch

    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(7)
    for hd, P in ((128, 16), (80, 16)):
        H, Hkv, lengths = 8, 2, [60, 70, 50]
        kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
        q = rng.integers(-(1 << 18), 1 << 18, size=(3, H * hd), dtype=np.int64)
        want = po.attention(q, kp, vp, table, lengths, 16, 0, None, None, 0)
        for bad in (-1, table.shape[1] * P + 1, 2 ** 31 - 1):
            device.read_flags()
            got = attend(q, kp, vp, table, [60, bad, 50])
            assert device.read_flags() == 16
            assert np.array_equal(got[[0, 2]], want[[0, 2]]) and not got[1].any()
            picked = device.paged_select(dev(q), torch.zeros((kp.shape[0], Hkv, 2, hd), dtype=torch.int32, device="cuda"), dev(table), dev(np.array([60, bad, 50], np.int32)), P, 3)
            assert device.read_flags() == 16 and (picked[1] == -1).all() and (picked[0, :, 0] == 0).all()
        assert np.array_equal(attend(q, kp, vp, table, [60, 70, 50], max_length=70), want)
        attend(q, kp, vp, table, [60, 70, 50], max_length=69)
        assert device.read_flags() == 16
        cos, sin = tables(65, hd, 16)                                   # no row for the token at 69
        got = attend(q, kp, vp, table, [60, 70, 50], cos=cos, sin=sin, rope=1)
        assert device.read_flags() == 16 and not got[1].any()
        for page in (-1, kp.shape[0], 2 ** 31 - 1):
            broken = table.copy()
            broken[1, 2] = page
            got = attend(q, kp, vp, broken, lengths)
            assert device.read_flags() == 16 and np.array_equal(got[[0, 2]], want[[0, 2]])
        pages = np.zeros((3, Hkv, 2), np.int32)
        pages[1, 0, 1] = table.shape[1]
        attend(q, kp, vp, table, lengths, pages=pages)
        assert device.read_flags() == 16
        # an append beyond the table, on a page outside the pool, beyond the rotation, a value beyond int32
        k = rng.integers(-(1 << 18), 1 << 18, size=(3, Hkv * hd), dtype=np.int64)
        for start, broken, kw in (([61, table.shape[1] * P, 51], table, {}), ([61, 2 ** 31 - 1, 51], table, {}), ([61, 0, 51], np.where(np.arange(len(table[0])) == 0, kp.shape[0], table), {}),
                                  ([1, 65, 2], table, dict(cos=dev(cos), sin=dev(sin), rope=1))):
            dkp, dvp = dev(kp), dev(vp)
            device.paged_append(dev(k), dev(k), dkp, dvp, dev(broken), dev(np.array(start, np.int32)), **kw)
            assert device.read_flags() == 16
        dkp, dvp = dev(kp), dev(vp)
        rows = np.array([0, 2, 1, 3], np.int32)                         # not ascending
        device.paged_append(dev(k), dev(k), dkp, dvp, dev(table), dev(np.array([0, 0, 0], np.int32)), rows=dev(rows))
        assert device.read_flags() == 16
        k[1, 3] = 1 << 31
        device.paged_append(dev(k), dev(k), dev(kp), dev(vp), dev(table), dev(np.array([59, 69, 49], np.int32)))
        assert device.read_flags() == 4


def test_flags_wait_for_the_default_stream():
    import torch

    from integer_inference_engine_b200 import device
    k = torch.zeros((1, 64), dtype=torch.int64, device="cuda")
    pages, table = torch.zeros((2, 1, 16, 64), dtype=torch.int32, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    inside, outside = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (3, 40))
    busy = torch.zeros((4096, 4096), device="cuda")
    device.paged_append(k, k, pages, pages.clone(), table, inside)
    device.read_flags()
    for _ in range(3):
        for _ in range(20):
            busy = busy @ busy                     # some milliseconds in front of the call whose flag is read
        device.paged_append(k, k, pages, pages, table, outside)
        assert device.read_flags() == 16 and device.read_flags() == 0


def test_no_sequences():
    import torch

    from integer_inference_engine_b200 import device
    z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device="cuda")
    pages = z(4, 2, 16, 64)
    assert device.paged_attention(z(0, 256, dtype=torch.int64), pages, pages, z(0, 3), z(0)).shape == (0, 256)
    assert device.paged_select(z(0, 256, dtype=torch.int64), z(4, 2, 2, 64), z(0, 3), z(0), 16, 4).shape == (0, 2, 4)
    device.paged_append(z(0, 128, dtype=torch.int64), z(0, 128, dtype=torch.int64), pages.clone(), pages.clone(), z(0, 3), z(0))
    assert device.read_flags() == 0


def step_world(rng, B, Hkv, hd, P, room, first):
    """A pool for B sequences with room for `room` positions each, their rows so far, and a contiguous copy."""
    import torch
    per = (room + P - 1) // P
    table = rng.permutation(B * per + 2)[:B * per].reshape(B, per).astype(np.int32)
    kp, vp = (torch.zeros((B * per + 2, Hkv, P, hd), dtype=torch.int32, device="cuda") for _ in range(2))
    bounds = torch.zeros((B * per + 2, Hkv, 2, hd), dtype=torch.int32, device="cuda")
    rows = [rng.integers(-(1 << 17), 1 << 17, size=(2, n, Hkv * hd), dtype=np.int64) for n in first]
    return kp, vp, bounds, table, rows


@pytest.mark.parametrize(("H", "Hkv", "hd", "P", "rope", "window"), [(8, 2, 128, 16, 1, 0), (8, 4, 64, 32, 2, 50), (4, 4, 128, 5, 1, 0)])
def test_prompts_and_steps_as_with_contiguous_caches(H, Hkv, hd, P, rope, window):
    """Prompts of different lengths go in as one packed batch, then steps of one token each: the bytes of attention_decode over contiguous
    caches, and with every page selected the same again."""
    import torch

    from integer_inference_engine_b200 import device
    from integer_inference_engine_b200.model import rope_tables
    rng = np.random.default_rng(P + hd)
    first, room = [60, 3, 0, 131], 150
    B = len(first)
    kp, vp, bounds, table, rows = step_world(rng, B, Hkv, hd, P, room, first)
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(room, hd, 50000.0, 16))
    turn = dict(cos=cos, sin=sin, rope=rope)
    table_d = dev(table)
    cu = dev(np.concatenate([[0], np.cumsum(first)]).astype(np.int32))
    k0, v0 = (dev(np.concatenate([r[i] for r in rows])) for i in (0, 1))
    device.paged_append(k0, v0, kp, vp, table_d, dev(np.zeros(B, np.int32)), rows=cu, bounds=bounds, **turn)
    caches = []
    for b, n in enumerate(first):
        kc, vc = (torch.zeros((Hkv, room, hd), dtype=torch.int32, device="cuda") for _ in range(2))
        if n:
            device.attention_prefill(torch.zeros((n, H * hd), dtype=torch.int64, device="cuda"), dev(rows[b][0]), dev(rows[b][1]), kc, vc, 0, H, Hkv, hd, **turn)
        caches.append((kc, vc))
    for step in range(6):
        q, k, v = (dev(rng.integers(-(1 << 17), 1 << 17, size=(B, n * hd), dtype=np.int64)) for n in (H, Hkv, Hkv))
        start = dev(np.array([n + step for n in first], np.int32))
        device.paged_append(k, v, kp, vp, table_d, start, bounds=bounds, **turn)
        lengths = start + 1
        got = device.paged_attention(q, kp, vp, table_d, lengths, window=window, **turn)
        every = device.paged_select(q, bounds, table_d, lengths, P, table.shape[1], window=window, **turn)
        again = device.paged_attention(q, kp, vp, table_d, lengths, window=window, pages=every, **turn)
        for b, (kc, vc) in enumerate(caches):
            want = device.attention_decode(q[b], k[b], v[b], kc, vc, first[b] + step, H, Hkv, hd, window=window, **turn)
            assert torch.equal(got[b], want), (step, b)
        assert torch.equal(again, got)
    assert device.read_flags() == 0


def test_a_whole_step_with_its_products_captured_and_replayed():
    """Q/K/V product, append, selection, attention and O product of a block as one graph over growing sequences, against the same calls made one
    by one; the positions are read on the device."""
    import torch

    from integer_inference_engine_b200 import device, qk_cuda, synth
    from integer_inference_engine_b200.model import rope_tables
    H, Hkv, hd, P, B, room, d = 8, 2, 128, 16, 3, 400, 512
    rng = np.random.default_rng(3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    wqkv = device.register_weight(synth.synth_q4k((H + 2 * Hkv) * hd * (d // 256), gen, 2e-4).view(-1), (H + 2 * Hkv) * hd, d // 256, qk_cuda.Q4_K)
    wo = device.register_weight(synth.synth_q4k(d * (H * hd // 256), gen, 2e-4).view(-1), d, H * hd // 256, qk_cuda.Q4_K)
    first = [200, 31, 17]
    kp, vp, bounds, table, rows = step_world(rng, B, Hkv, hd, P, room, first)
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(room, hd, 50000.0, 16))
    turn = dict(cos=cos, sin=sin, rope=1)
    table_d, cu = dev(table), dev(np.concatenate([[0], np.cumsum(first)]).astype(np.int32))
    device.paged_append(*(dev(np.concatenate([r[i] for r in rows])) for i in (0, 1)), kp, vp, table_d, dev(np.zeros(B, np.int32)), rows=cu, bounds=bounds, **turn)
    xs = [dev(rng.integers(-(1 << 17), 1 << 17, size=(B, d), dtype=np.int64)) for _ in range(5)]

    def step(x, start, lengths, kp, vp, bounds):
        qkv = device.apply(wqkv, x, (H + 2 * Hkv) * hd, 24)
        q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + Hkv) * hd], qkv[:, (H + Hkv) * hd:]
        device.paged_append(k, v, kp, vp, table_d, start, bounds=bounds, **turn)
        pages = device.paged_select(q, bounds, table_d, lengths, P, 4, **turn)
        att = device.paged_attention(q, kp, vp, table_d, lengths, pages=pages, **turn) + device.paged_attention(q, kp, vp, table_d, lengths, **turn)
        return device.apply(wo, att, d, 24)

    want, mine = [], [t.clone() for t in (kp, vp, bounds)]
    start = dev(np.array(first, np.int32))
    for i, x in enumerate(xs):
        want.append(step(x, start + i, start + i + 1, *mine))
    cell, at, n = xs[0].clone(), start.clone(), start + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    scratch = [t.clone() for t in (kp, vp, bounds)]
    with torch.cuda.stream(side):
        step(cell, at, n, *scratch)                                     # workspaces of the products
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cell, at, n, kp, vp, bounds)
    for x, w in zip(xs, want):
        cell.copy_(x)
        graph.replay()
        assert torch.equal(out, w)
        at += 1
        n += 1
    assert all(torch.equal(a, b) for a, b in zip((kp, vp, bounds), mine)) and device.read_flags() == 0
    qk_cuda.free_all()


def test_calls_on_two_streams_share_nothing():
    import torch

    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(1)
    H, Hkv, hd, P, lengths = 8, 2, 128, 16, [900, 40, 333]
    worlds = []
    for i in range(2):
        kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
        q = rng.integers(-(1 << 18), 1 << 18, size=(3, H * hd), dtype=np.int64)
        worlds.append([dev(t) for t in (q, kp, vp, table, np.array(lengths, np.int32))] + [po.attention(q, kp, vp, table, lengths, 16, 0, None, None, 0)])
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in worlds], [[], []]
    for _ in range(20):
        for i, (w, s) in enumerate(zip(worlds, streams)):
            with torch.cuda.stream(s):
                outs[i].append(device.paged_attention(*w[:5]))
    torch.cuda.synchronize()
    for w, got in zip(worlds, outs):
        assert all(np.array_equal(g.cpu().numpy(), w[5]) for g in got)


def test_a_long_cache_whose_offsets_pass_32_bits():
    """Pages beyond 2^31 values: the last ones of a pool of nine gigabytes hold the keys."""
    import torch

    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(5)
    H, Hkv, hd, P, n = 8, 2, 128, 16, 100
    n_pages = (1 << 31) // (Hkv * P * hd) + 40
    try:
        kp, vp = (torch.empty((n_pages, Hkv, P, hd), dtype=torch.int32, device="cuda") for _ in range(2))
    except torch.cuda.OutOfMemoryError:
        pytest.skip("not enough memory")
    table = (n_pages - 1 - np.arange(7, dtype=np.int32))[None]
    k, v = (rng.integers(-(1 << 18), 1 << 18, size=(n, Hkv * hd), dtype=np.int64) for _ in range(2))
    device.paged_append(dev(k), dev(v), kp, vp, dev(table), dev(np.zeros(1, np.int32)), rows=dev(np.array([0, n], np.int32)))
    q = rng.integers(-(1 << 18), 1 << 18, size=(1, H * hd), dtype=np.int64)
    got = device.paged_attention(dev(q), kp, vp, dev(table), dev(np.array([n], np.int32))).cpu().numpy()
    small_k, small_v = (np.zeros((7, Hkv, P, hd), np.int32) for _ in range(2))
    po.append(k, v, small_k, small_v, np.zeros((7, Hkv, 2, hd), np.int32), np.arange(7)[None], [0], [0, n], 16, None, None, 0)
    assert np.array_equal(got, po.attention(q, small_k, small_v, np.arange(7)[None], [n], 16, 0, None, None, 0))
    assert device.read_flags() == 0
    del kp, vp
    torch.cuda.empty_cache()
