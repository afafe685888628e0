"""The paged key/value cache at the ends of what its entries accept: the largest head dimensions, tables, lists, what lies half outside the cache.
Every result is equal, bit for bit, to the restatement in NumPy's 64-bit integers."""
import numpy as np
import pytest

from oracle import paged_oracle as po
from test_gpu_paged import attend, dev, pool, tables

pytestmark = pytest.mark.gpu


def appended(rng, P, Hkv, hd, k, v, table, start, rows, rope_rows, counts):
    """What an append leaves (keys, values, bounds, flags), and what it should where sequence i takes counts[i] rows from rows[i] on."""
    from integer_inference_engine_b200 import device
    kp, vp = (rng.integers(-(1 << 18), 1 << 18, size=(int(table.max()) + 3, Hkv, P, hd)).astype(np.int32) for _ in range(2))
    bounds = rng.integers(-9, 9, size=(kp.shape[0], Hkv, 2, hd)).astype(np.int32)
    cos, sin = tables(rope_rows, hd, 16)
    dkp, dvp, db = dev(kp), dev(vp), dev(bounds)
    device.read_flags()
    device.paged_append(dev(k), dev(v), dkp, dvp, dev(table), dev(np.array(start, np.int32)), rows=None if rows is None else dev(np.array(rows, np.int32)), cos=dev(cos), sin=dev(sin), rope=1, bounds=db)
    flags = device.read_flags()
    for b, n in enumerate(counts):                 # (each by itself: the restatement knows no rows that are left out)
        at = b if rows is None else rows[b]
        if n > 0:
            po.append(k[at:at + n], v[at:at + n], kp, vp, bounds, table[b:b + 1], start[b:b + 1], [0, n], 16, cos, sin, 1)
    return [t.cpu().numpy() for t in (dkp, dvp, db)], [kp, vp, bounds], flags


@pytest.mark.parametrize(("P", "start", "counts", "inside"), [
    (16, [16, 2], [7, 3], [4, 3]),                 # positions 20, 21 and 22 lie behind the table of rotations, within a page that begins in front of them
    (16, [3, 0], [30, 5], [17, 5]),                # ... and in the next pages
    (32, [19, 20], [2, 1], [1, 0]),
    (5, [18, 25], [4, 2], [2, 0]),
])
def test_rows_in_front_of_the_rotation_tables_end_are_appended(P, start, counts, inside):
    rng = np.random.default_rng(P + start[0])
    Hkv, hd, rows = 2, 32, [0] + list(np.cumsum(counts))
    per = 40 // P + 2
    table = rng.permutation(2 * per).reshape(2, per).astype(np.int32)
    k, v = (rng.integers(-(1 << 18), 1 << 18, size=(sum(counts), Hkv * hd), dtype=np.int64) for _ in range(2))
    got, want, flags = appended(rng, P, Hkv, hd, k, v, table, start, rows, 20, inside)
    assert flags == 16
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("P", [1, 4])
@pytest.mark.parametrize("wrong", [1, 127, 128, 200, 299])
@pytest.mark.parametrize("how", ["descends", "passes the end"])
def test_wrong_rows_of_any_sequence_are_flagged(P, wrong, how):
    """More sequences than a scan takes at once: the wrong one gets no rows, the others theirs (as long as there are no more of
    these than rows: eight lie behind the last sequence's)."""
    rng = np.random.default_rng(wrong + P)
    B, Hkv, hd, each = 300, 1, 16, 2
    rows = [i * each for i in range(B + 1)]
    counts = [each] * B
    if how == "descends":
        if wrong == B - 1:
            rows[B] = rows[B - 1] - 1
        else:
            rows[wrong + 1] = rows[wrong] - 1      # the one behind begins in front of it
            counts[wrong + 1] = rows[wrong + 2] - rows[wrong + 1]
        counts[wrong] = 0
    elif wrong == B - 1:
        rows[B] += 9
        counts[wrong] = 0
    else:
        rows[wrong + 1] = B * each + 9             # beyond all rows: the one behind descends
        counts[wrong] = counts[wrong + 1] = 0
    table = rng.permutation(B * 6).reshape(B, 6).astype(np.int32)
    k, v = (rng.integers(-(1 << 18), 1 << 18, size=(B * each + 8, Hkv * hd), dtype=np.int64) for _ in range(2))
    got, want, flags = appended(rng, P, Hkv, hd, k, v, table, [0] * B, rows, 40, counts)
    assert flags == 16
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize(("hd", "P"), [(128, 16), (80, 16), (64, 5)])
@pytest.mark.parametrize("window", [0, 4])
def test_lengths_beyond_a_bound_of_zero_are_flagged(hd, P, window):
    """max_length = 0: no sequence has a key, one that says otherwise is left out."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(hd)
    H, Hkv = 4, 2
    kp, vp, table = pool(rng, [30, 20], P, Hkv, hd, 18)
    q = rng.integers(-(1 << 18), 1 << 18, size=(2, H * hd), dtype=np.int64)
    for lengths, flags in (([0, 0], 0), ([0, 3], 16), ([-1, 0], 16)):
        device.read_flags()
        got = attend(q, kp, vp, table, lengths, max_length=0, window=window)
        assert device.read_flags() == flags and not got.any()


@pytest.mark.parametrize("hd", [768, 770, 1024])
@pytest.mark.parametrize("chosen", [False, True])
def test_attention_of_large_heads(hd, chosen):
    """Eight query heads of these are 48 KB as 64 bits, the first size beyond it, and the largest that is accepted; more than eight heads a KV head."""
    from integer_inference_engine_b200 import device
    H, Hkv, P, lengths = 9, 1, 16, [40, 0, 3]
    rng = np.random.default_rng(hd)
    kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
    q = rng.integers(-(1 << 18), 1 << 18, size=(len(lengths), H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    pages = np.array([[[2, 0]], [[0, 1]], [[-1, 0]]], np.int32) if chosen else None
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=2, pages=pages)
    assert device.read_flags() == 0
    assert np.array_equal(got, po.attention(q, kp, vp, table, lengths, 16, 0, cos, sin, 2, pages))


# head dimension, query heads of a KV head (as many as its queries are padded to), pages of the table: queries, pages on their way and scores together pass 220 KB of shared memory
RANK = [(384, 4, 769), (384, 3, 1000), (352, 8, 1024), (304, 16, 1000), (240, 32, 1000), (48, 328, 1000), (384, 4, 768), (272, 24, 1000), (64, 240, 300)]


@pytest.mark.parametrize(("hd", "rep", "per"), RANK)
def test_select_of_large_heads_from_wide_tables(hd, rep, per):
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(hd + per)
    lengths, n_pages = [per - 1, 37, 0], 50
    bounds = np.sort(rng.integers(-(1 << 18), 1 << 18, size=(n_pages, 1, 2, hd)), axis=2)[:, :, ::-1].astype(np.int32)
    table = rng.integers(0, n_pages, size=(3, per)).astype(np.int32)
    q = rng.integers(-(1 << 18), 1 << 18, size=(3, rep * hd), dtype=np.int64)
    device.read_flags()
    got = device.paged_select(dev(q), dev(bounds), dev(table), dev(np.array(lengths, np.int32)), 1, 9)
    assert device.read_flags() == 0
    assert np.array_equal(got.cpu().numpy(), po.select(q, bounds, table, lengths, 1, 9, 1, 1, 16, 0, None, None, 0))


# heads, KV heads, lengths' bound, sequences (on 148 SMs: pairs dealt out whole, 305 tiles each; an even cut with whole pairs in it; pairs of 700 tiles cut into parts of some 300)
@pytest.mark.parametrize(("H", "Hkv", "most", "B"), [(8, 4, 39000, 37), (8, 8, 39000, 40), (8, 4, 89600, 16)])
def test_more_tiles_of_a_pair_than_one_accumulation_takes(H, Hkv, most, B):
    """Output sums are read out every 256 tiles of 128 keys.  Few physical pages stand behind all tables."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(B)
    hd, P, n_pages = 32, 16, 60
    lengths = [most] + [int(n) for n in most - rng.integers(0, 100, size=B - 1)]
    kp, vp = (rng.integers(-(1 << 18), 1 << 18, size=(n_pages, Hkv, P, hd)).astype(np.int32) for _ in range(2))
    vp[:, 0] = rng.choice(np.array([-(1 << 31), (1 << 31) - 1, -1], np.int64), size=vp[:, 0].shape)       # the largest sums that there are
    table = rng.integers(0, n_pages, size=(B, (most + P - 1) // P)).astype(np.int32)
    q = rng.integers(-(1 << 14), 1 << 14, size=(B, H * hd), dtype=np.int64)
    cos, sin = tables(most, hd, 16)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=1)
    assert device.read_flags() == 0
    for b in (0, 1, B // 2, B - 1):
        assert np.array_equal(got[b:b + 1], po.attention(q[b:b + 1], kp, vp, table[b:b + 1], lengths[b:b + 1], 16, 0, cos, sin, 1)), b


@pytest.mark.parametrize(("H", "Hkv", "hd", "lengths"), [(12, 1, 128, [5000, 3000]), (20, 1, 64, [9000]), (32, 2, 96, [4000, 0, 7000, 100]), (9, 1, 32, [20000, 1])])
def test_more_than_eight_heads_over_a_long_cache(H, Hkv, hd, lengths):
    """Several groups of query heads per KV head, their pairs cut between CTAs."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(H)
    kp, vp, table = pool(rng, lengths, 16, Hkv, hd, 18)
    q = rng.integers(-(1 << 16), 1 << 16, size=(len(lengths), H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=2)
    assert device.read_flags() == 0
    assert np.array_equal(got, po.attention(q, kp, vp, table, lengths, 16, 0, cos, sin, 2))


@pytest.mark.parametrize("hd", [64, 80])
@pytest.mark.parametrize("chosen", [False, True])
def test_scratch_in_parts(hd, chosen):
    """Tables (or lists) so wide that the scratch of all sequences passes its limit: they go in parts, one behind the other, over the same scratch."""
    import torch

    from integer_inference_engine_b200 import device, qk_cuda
    H, Hkv, P, per = 8, 2, 16, 2048
    size = lambda n: qk_cuda.load_library().iie_paged_attn_bytes(n, per * P, 0, per if chosen else 0, P, H, Hkv, hd, 16)
    part = (2 << 30) // size(1)
    B = part + 37
    assert size(B) == size(part) > 1 << 29
    rng = np.random.default_rng(hd)
    lengths = [int(n) for n in rng.integers(0, 41, size=B)]
    lengths[part - 1:part + 1] = [600, 500]        # the last of a part, the first of the next
    kp, vp, narrow = pool(rng, lengths, P, Hkv, hd, 18)
    table = np.full((B, per), -7, np.int32)
    table[:, :narrow.shape[1]] = narrow
    pages = None
    if chosen:
        pages = np.full((B, Hkv, per), -1, np.int32)
        for b, n in enumerate(lengths):
            take = rng.permutation((n + P - 1) // P)[:20]
            for g in range(Hkv):
                pages[b, g, rng.permutation(per)[:len(take)]] = take
    q = rng.integers(-(1 << 18), 1 << 18, size=(B, H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    device.read_flags()
    got = attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=1, pages=pages)
    torch.cuda.empty_cache()
    assert device.read_flags() == 0
    assert np.array_equal(got, po.attention(q, kp, vp, table, lengths, 16, 0, cos, sin, 1, pages))


@pytest.mark.parametrize(("H", "Hkv", "hd", "lengths"), [(32, 4, 128, [300]), (32, 8, 128, [1500, 0, 700, 1100]), (8, 2, 64, [40] * 30), (4, 2, 80, [90, 3])])
def test_a_table_with_room_for_much_more(H, Hkv, hd, lengths):
    """2048 pages a sequence, whatever its length, entries behind its last page pointing nowhere: attention, selection, attention over what it selects."""
    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(hd + len(lengths))
    P, B = 16, len(lengths)
    kp, vp, narrow = pool(rng, lengths, P, Hkv, hd, 18)
    table = np.full((B, 2048), -7, np.int32)
    table[:, :narrow.shape[1]] = narrow
    bounds = np.stack([kp.max(2), kp.min(2)], 2)
    q = rng.integers(-(1 << 17), 1 << 17, size=(B, H * hd), dtype=np.int64)
    cos, sin = tables(max(lengths), hd, 16)
    device.read_flags()
    assert np.array_equal(attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=1), po.attention(q, kp, vp, table, lengths, 16, 0, cos, sin, 1))
    pages = device.paged_select(dev(q), dev(bounds), dev(table), dev(np.array(lengths, np.int32)), P, 6, cos=dev(cos), sin=dev(sin), rope=1).cpu().numpy()
    assert np.array_equal(pages, po.select(q, bounds, table, lengths, P, 6, 1, 1, 16, 0, cos, sin, 1))
    assert np.array_equal(attend(q, kp, vp, table, lengths, cos=cos, sin=sin, rope=1, pages=pages), po.attention(q, kp, vp, table, lengths, 16, 0, cos, sin, 1, pages))
    assert device.read_flags() == 0


def test_two_captured_steps_replayed_at_once():
    """Selection, attention over it and over everything, captured twice and replayed on two streams: neither graph's scratch is the other's."""
    import torch

    from integer_inference_engine_b200 import device
    rng = np.random.default_rng(3)
    H, Hkv, hd, P, lengths = 8, 2, 128, 16, [900, 40, 3000]
    graphs, outs, wants, streams = [], [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        kp, vp, table = pool(rng, lengths, P, Hkv, hd, 18)
        bounds = np.stack([kp.max(2), kp.min(2)], 2)
        q = rng.integers(-(1 << 17), 1 << 17, size=(3, H * hd), dtype=np.int64)
        world = [dev(t) for t in (q, kp, vp, table, np.array(lengths, np.int32), bounds)]
        pages = po.select(q, bounds, table, lengths, P, 8, 1, 1, 16, 0, None, None, 0)
        wants.append([pages] + [po.attention(q, kp, vp, table, lengths, 16, 0, None, None, 0, p) for p in (pages, None)])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            picked = device.paged_select(world[0], world[5], world[3], world[4], P, 8)
            outs.append([picked, device.paged_attention(*world[:5], pages=picked), device.paged_attention(*world[:5])])
        graphs.append((graph, world))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, wants):
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want))
    assert device.read_flags() == 0

