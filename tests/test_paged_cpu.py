"""What the paged cache's entries refuse, without a GPU: arguments are looked at before anything is launched."""
import pytest
import torch

from integer_inference_engine_b200 import build, device, qk_cuda

I32, I64 = torch.int32, torch.int64


@pytest.fixture(scope="module")
def lib():
    build.build()
    return qk_cuda.load_library()


def good():
    """Arguments that stand: 3 sequences, 4 heads over 2 KV heads of 64, pages of 16 rows."""
    z = lambda *shape, dtype=I32: torch.zeros(shape, dtype=dtype)
    return dict(kpages=z(9, 2, 16, 64), vpages=z(9, 2, 16, 64), table=z(3, 5), lengths=z(3), start=z(3), q=z(3, 256, dtype=I64), k=z(3, 128, dtype=I64), v=z(3, 128, dtype=I64),
                bounds=z(9, 2, 2, 64), cos=z(80, 32, dtype=I64), sin=z(80, 32, dtype=I64), pages=z(3, 2, 2))


def call(name, w, **kw):
    if name == "append":
        return device.paged_append(w["k"], w["v"], w["kpages"], w["vpages"], w["table"], w["start"], bounds=w["bounds"], **kw)
    if name == "attention":
        return device.paged_attention(w["q"], w["kpages"], w["vpages"], w["table"], w["lengths"], pages=w["pages"], **kw)
    return device.paged_select(w["q"], w["bounds"], w["table"], w["lengths"], kw.pop("page_rows", 16), kw.pop("n_select", 4), **kw)


REFUSED = [
    ("append", dict(kpages=torch.zeros(9, 2, 16, 64, dtype=I64)), {}), ("append", dict(vpages=torch.zeros(9, 2, 16, 32, dtype=I32)), {}),
    ("append", dict(kpages=torch.zeros(9, 16, 2, 64, dtype=I32).transpose(1, 2)), {}), ("append", dict(kpages=torch.zeros(0, 2, 16, 64, dtype=I32), vpages=torch.zeros(0, 2, 16, 64, dtype=I32)), {}),
    ("append", dict(table=torch.zeros(3, 5, dtype=I64)), {}), ("append", dict(table=torch.zeros(3, 10, dtype=I32)[:, ::2]), {}), ("append", dict(table=torch.zeros(3, 0, dtype=I32)), {}),
    ("append", dict(start=torch.zeros(4, dtype=I32)), {}), ("append", dict(start=torch.zeros(3, dtype=I64)), {}), ("append", dict(start=torch.zeros(6, dtype=I32)[::2]), {}),
    ("append", dict(k=torch.zeros(3, 128)), {}), ("append", dict(v=torch.zeros(3, 128, dtype=I32)), {}), ("append", dict(k=torch.zeros(3, 64, dtype=I64), v=torch.zeros(3, 64, dtype=I64)), {}),
    ("append", dict(k=torch.zeros(2, 128, dtype=I64), v=torch.zeros(2, 128, dtype=I64)), {}), ("append", dict(k=torch.zeros(128, 3, dtype=I64).T), {}),
    ("append", dict(k=torch.zeros(1, 128, dtype=I64).expand(3, 128)), {}),
    ("append", {}, dict(rows=torch.zeros(3, dtype=I32))), ("append", {}, dict(rows=torch.zeros(4, dtype=I64))), ("append", dict(bounds=torch.zeros(9, 2, 64, 2, dtype=I32)), {}),
    ("append", {}, dict(rope=3)), ("append", {}, dict(rope=1)), ("append", {}, dict(rope=1, cos=torch.zeros(80, 32, dtype=I64), sin=torch.zeros(79, 32, dtype=I64))),
    ("append", {}, dict(rope=2, cos=torch.zeros(80, 64, dtype=I64), sin=torch.zeros(80, 64, dtype=I64))),
    ("attention", dict(q=torch.zeros(3, 256, dtype=I32)), {}), ("attention", dict(q=torch.zeros(2, 256, dtype=I64)), {}), ("attention", dict(q=torch.zeros(3, 192, dtype=I64)), {}),
    ("attention", dict(q=torch.zeros(256, 3, dtype=I64).T), {}), ("attention", dict(lengths=torch.zeros(2, dtype=I32)), {}), ("attention", dict(pages=torch.zeros(3, 2, 0, dtype=I32)), {}),
    ("attention", dict(pages=torch.zeros(3, 1, 2, dtype=I32)), {}), ("attention", dict(pages=torch.zeros(3, 2, 2, dtype=I64)), {}), ("attention", {}, dict(max_length=81)),
    ("attention", {}, dict(max_length=-1)), ("attention", {}, dict(window=-1)), ("attention", {}, dict(out=torch.zeros(3, 255, dtype=I64))), ("attention", {}, dict(out=torch.zeros(3, 256, dtype=I32))),
    ("attention", {}, dict(out=torch.zeros(256, 3, dtype=I64).T)), ("attention", {}, dict(rope=1)), ("attention", dict(kpages=torch.zeros(9, 2, 16, 64)), {}),
    ("select", dict(bounds=torch.zeros(9, 2, 64, 2, dtype=I32)), {}), ("select", dict(bounds=torch.zeros(9, 2, 2, 64, dtype=I64)), {}), ("select", {}, dict(n_select=0)), ("select", {}, dict(page_rows=0)),
    ("select", {}, dict(keep_first=3, keep_last=2)), ("select", {}, dict(keep_first=-1)), ("select", {}, dict(window=-5)), ("select", {}, dict(out=torch.zeros(3, 2, 5, dtype=I32))),
    ("select", dict(q=torch.zeros(3, 100, dtype=I64)), {}), ("select", dict(lengths=torch.zeros(3, dtype=I64)), {}),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refused(case):
    name, change, kw = REFUSED[case]
    with pytest.raises(ValueError):
        call(name, {**good(), **change}, **dict(kw))


def test_an_output_over_the_queries_is_refused():
    """In place, one row on, and as columns of the matrix that holds the queries; beside them the path is taken (and finds no GPU, or tensors of another device)."""
    w, wide = good(), torch.zeros(4, 256, dtype=I64)
    for q, out in ((wide[:3], wide[:3]), (wide[:3], wide[1:]), (wide[1:], wide[:3])):
        with pytest.raises(ValueError, match="overlap"):
            call("attention", {**w, "q": q}, out=out)
    both = torch.zeros(6, 256, dtype=I64)
    with pytest.raises((ValueError, qk_cuda.CudaUnavailableError)) as e:
        call("attention", {**w, "q": both[:3]}, out=both[3:])
    assert "overlap" not in str(e.value)


@pytest.mark.parametrize("name", ["append", "attention", "select"])
def test_tensors_of_another_device_are_refused(name):
    """Good arguments on the CPU: without a GPU there is no path, with one they lie on the wrong device."""
    with pytest.raises((ValueError, qk_cuda.CudaUnavailableError)):
        call(name, good(), rope=1, cos=good()["cos"], sin=good()["sin"])


def test_scratch_of_attention(lib):
    size = lib.iie_paged_attn_bytes
    assert 0 < size(1, 300, 0, 0, 16, 32, 4, 128, 16) < size(1, 4096, 0, 0, 16, 32, 4, 128, 16)
    assert size(8, 32000, 2048, 0, 16, 32, 4, 128, 16) < size(8, 32000, 0, 0, 16, 32, 4, 128, 16)
    assert size(1000, 100000, 0, 0, 16, 32, 4, 128, 16) < 6 << 30                # parts behind one another
    for bad in ((-1, 10, 0, 0, 16, 4, 2, 64, 16), (1, -1, 0, 0, 16, 4, 2, 64, 16), (1, 10, 0, -1, 16, 4, 2, 64, 16), (1, 10, 0, 0, 0, 4, 2, 64, 16), (1, 10, 0, 0, 16, 5, 2, 64, 16), (1, 10, 0, 0, 16, 4, 2, 63, 16), (1, 10, 0, 0, 16, 4, 2, 64, 0),
                (1, 10, 0, 1 << 30, 16, 4, 2, 64, 16), (70000, 10, 0, 0, 16, 4, 2, 64, 16)):
        assert size(*bad) == -1, bad


def test_c_entries_refuse(lib):
    """Status 1 before any pointer is looked at."""
    append = lambda **c: lib.iie_paged_append_dev(*{**dict(k=None, v=None, narrow=0, k_ld=128, v_ld=128, tokens=3, kp=None, vp=None, n_pages=9, P=16, table=None, ld=5, start=None, rows=None, B=3, cos=None,
                                                        sin=None, rr=0, rope=0, kv=2, hd=64, fa=16, bounds=None, stream=None), **c}.values())
    assert append() == 1                                                     # null pointers
    for c in (dict(k_ld=127), dict(v_ld=0), dict(tokens=-1), dict(tokens=2), dict(n_pages=0), dict(P=0), dict(ld=0), dict(B=-1), dict(rope=1), dict(rope=4), dict(hd=63), dict(hd=0), dict(fa=0), dict(fa=30), dict(kv=0),
              dict(ld=1 << 30)):
        assert append(**c) == 1, c
    assert append(B=0) == 0
    attn = lambda **c: lib.iie_paged_attn_dev(*{**dict(q=None, q_ld=256, kp=None, vp=None, n_pages=9, P=16, table=None, ld=5, lengths=None, B=3, max_length=80, sel=None, n_sel=0, window=0, cos=None, sin=None, rr=0,
                                                    rope=0, H=4, kv=2, hd=64, fa=16, inv=8192, work=None, bytes=1 << 30, out=None, stream=None), **c}.values())
    assert attn() == 1
    for c in (dict(q_ld=255), dict(max_length=81), dict(n_sel=2), dict(H=5), dict(rope=2), dict(fa=31), dict(bytes=0), dict(max_length=-1), dict(n_pages=1 << 29), dict(work=8), dict(kp=4), dict(vp=1)):
        assert attn(**c) == 1, c
    assert attn(B=0) == 0
    select = lambda **c: lib.iie_paged_select_dev(*{**dict(q=None, q_ld=256, bounds=None, n_pages=9, P=16, table=None, ld=5, lengths=None, B=3, n=4, first=1, last=1, window=0, cos=None, sin=None, rr=0, rope=0, H=4,
                                                        kv=2, hd=64, fa=16, score=None, out=None, stream=None), **c}.values())
    assert select() == 1
    for c in (dict(n=0), dict(first=4), dict(last=-1), dict(H=3), dict(q_ld=1), dict(hd=0)):
        assert select(**c) == 1, c
    assert select(B=0) == 0


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 4])
def test_counts_beyond_31_bits_are_refused(n):
    """... before they are cut to the 32 bits that the library takes, and before anything of that size is laid out."""
    with pytest.raises(ValueError, match="n_select"):
        call("select", good(), n_select=n)
    with pytest.raises(ValueError, match="rows of a sequence"):
        call("attention", {**good(), "pages": torch.empty((3, 2, n), dtype=I32, device="meta")})
