"""The paged-cache C ABI without a GPU: declarations, struct layouts, and the refusals that come before any device work."""
import ctypes
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "s2d_cache.h").read_text(), flags=re.S)


@pytest.fixture(scope="module")
def kv():
    from fish_s2pro_b200 import build, kvcache
    build.build_runtime()
    return kvcache


def test_bindings_match_the_header(kv):
    counts = {n: p.count(",") + 1 for n, p in re.findall(r"\b(s2d_cache_\w+)\s*\(([^;{]*?)\)\s*;", HEADER, flags=re.S)}
    assert sorted(counts) == sorted(kv.CACHE_SIGNATURES)
    for name, n in counts.items():
        assert hasattr(kv.cache_lib(), name) and len(kv.CACHE_SIGNATURES[name][1]) == n


@pytest.mark.parametrize("name,cls", [("S2dCacheView", "_View"), ("S2dCacheAppend", "_Append"), ("S2dCacheAttention", "_Attention"),
                                      ("S2dCacheEvict", "_Evict")])
def test_structs_match_the_header(kv, name, cls):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    fields = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            base, names = re.match(r"(?:const )?(\w+) (.*)", decl, re.S).groups()
            fields += [(n.strip().lstrip("*").strip(), "ptr" if "*" in n else base) for n in names.split(",")]
    kinds = {"ptr": ctypes.c_void_p, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "double": ctypes.c_double,
             "size_t": ctypes.c_size_t}
    assert [(n, kinds[t]) for n, t in fields] == list(getattr(kv, cls)._fields_)


def test_constants_match_the_header(kv):
    c = {n: int(v) for n, v in re.findall(r"#define (S2D_\w+) (\d+)", HEADER)}
    assert c["S2D_CACHE_PAGE"] == kv.PAGE
    assert (c["S2D_CACHE_BAD_PAGE"], c["S2D_CACHE_BAD_LENGTH"], c["S2D_CACHE_FULL"], c["S2D_CACHE_ABORTED"]) == \
        (kv.BAD_PAGE, kv.BAD_LENGTH, kv.FULL, kv.ABORTED)
    assert (c["S2D_TYPE_F32"], c["S2D_TYPE_F16"], c["S2D_TYPE_BF16"]) == (0, 1, 30)


A = 0x10000  # an aligned address that nothing reads: every call below is refused, or computes sizes only


def view(kv, **kw):
    d = dict(k=A, v=A, page_stride=2 * 64 * 64, head_stride=64 * 64, page_table=A, table_stride=3, lengths=A, positions=A, mass=A, status=A,
             n_seq=2, kv_heads=2, head_dim=64, n_pages=6, max_pages=3, type=1, device=0)
    d.update(kw)
    return kv._View(**d)


def refused(kv, fn, v, a):
    err = ctypes.create_string_buffer(256)
    rc = getattr(kv.cache_lib(), fn)(ctypes.byref(v) if v is not None else None, ctypes.byref(a) if a is not None else None, None, err, 256)
    assert rc == -1 and err.value, (rc, err.value)
    return err.value.decode()


BAD_VIEWS = [dict(k=0), dict(v=0), dict(page_table=0), dict(lengths=0), dict(head_dim=96), dict(type=0), dict(type=8), dict(n_seq=0),
             dict(kv_heads=0), dict(n_pages=0), dict(max_pages=0), dict(n_seq=65536), dict(kv_heads=1025), dict(max_pages=2 ** 18 + 1, table_stride=2 ** 18 + 1),
             dict(table_stride=2), dict(head_stride=64 * 64 - 8), dict(head_stride=64 * 64 + 4, page_stride=2 ** 20), dict(page_stride=2 * 64 * 64 - 8),
             dict(page_stride=2 * 64 * 64 + 4), dict(k=A + 8), dict(v=A + 2)]


@pytest.mark.parametrize("bad", BAD_VIEWS)
def test_bad_views_are_refused(kv, bad):
    v = view(kv, **bad)
    refused(kv, "s2d_cache_append", v, append(kv))
    refused(kv, "s2d_cache_attention", v, attention(kv))
    refused(kv, "s2d_cache_evict", v, evict(kv))


def append(kv, **kw):
    d = dict(q=A, k=A, v=A, q_stride=256, k_stride=128, v_stride=128, q_out=A, q_out_stride=256, pos=A, past=A + 4096, tokens=2, heads=4, type=1,
             eps=1e-6, rope_base=1e6)
    d.update(kw)
    return kv._Append(**d)


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(q=0), dict(k=0), dict(v=0), dict(q_out=0), dict(pos=0), dict(past=0), dict(heads=0), dict(heads=3),
                                 dict(heads=34), dict(tokens=3), dict(type=30), dict(type=2), dict(q_stride=255), dict(k_stride=4), dict(v_stride=-128),
                                 dict(q=A + 8), dict(q_out=A + 2), dict(q_out_stride=128), dict(rope_base=0.0), dict(rope_base=float("inf")),
                                 dict(rope_base=float("nan")), dict(eps=-1.0), dict(eps=float("nan")), dict(past=A), dict(past=A + 4),
                                 dict(q_out=A + 16), dict(q_out=A + 1008, q_stride=512)])
def test_bad_appends_are_refused(kv, bad):
    refused(kv, "s2d_cache_append", view(kv), append(kv, **bad))


def attention(kv, **kw):
    d = dict(q=A, q_stride=256, out=A + 65536, out_stride=256, tokens=2, heads=4, type=1, scale=0.125)
    d.update(kw)
    return kv._Attention(**d)


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(q=0), dict(out=0), dict(heads=0), dict(heads=3), dict(heads=34), dict(tokens=3), dict(type=30),
                                 dict(type=12), dict(prefix_len=-1), dict(prefix_len=5), dict(prefix_len=2 ** 24 + 1, prefix_pages=A),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(q_stride=252), dict(out_stride=4), dict(q=A + 8),
                                 dict(out=A + 65538), dict(q_stride=-256), dict(out_stride=248), dict(out=A), dict(out=A + 512),
                                 dict(prefix_len=70, prefix_pages=A, workspace=0), dict(prefix_len=70, prefix_pages=A, workspace=A, workspace_bytes=16),
                                 dict(prefix_len=70, prefix_pages=A, workspace=A + 16, workspace_bytes=2 ** 30), dict(tokens=2 ** 25, heads=4, q_start=A)])
def test_bad_attentions_are_refused(kv, bad):
    refused(kv, "s2d_cache_attention", view(kv), attention(kv, **bad))


def test_weighing_needs_mass(kv):
    assert "mass" in refused(kv, "s2d_cache_attention", view(kv, mass=0), attention(kv, weigh=1))


def evict(kv, **kw):
    d = dict(budget=64, recent=8, past=A + 4096, workspace=A, workspace_bytes=2 ** 24)
    d.update(kw)
    return kv._Evict(**d)


@pytest.mark.parametrize("bad", [dict(budget=0), dict(budget=-3), dict(recent=-1), dict(recent=65), dict(past=A), dict(past=A + 4), dict(workspace=0),
                                 dict(workspace_bytes=16), dict(workspace=A + 64)])
def test_bad_evictions_are_refused(kv, bad):
    refused(kv, "s2d_cache_evict", view(kv), evict(kv, **bad))


def test_evicting_needs_positions_and_mass(kv):
    refused(kv, "s2d_cache_evict", view(kv, mass=0), evict(kv))
    refused(kv, "s2d_cache_evict", view(kv, positions=0), evict(kv))


@pytest.mark.parametrize("fn", ["s2d_cache_append", "s2d_cache_attention", "s2d_cache_evict"])
def test_null_structs_are_refused(kv, fn):
    refused(kv, fn, None, None)
    refused(kv, fn, view(kv), None)


def test_workspace_sizes(kv):
    """No workspace for a lone decode step; what a prefix or prompts need grows with the rows; alignment padding included."""
    L, n, err = kv.cache_lib(), ctypes.c_size_t(), ctypes.create_string_buffer(256)

    def size(**kw):
        assert L.s2d_cache_attention_workspace(ctypes.byref(view(kv)), ctypes.byref(attention(kv, **kw)), ctypes.byref(n), err, 256) == 0, err.value
        return n.value

    assert size() == 0
    one = size(prefix_len=70, prefix_pages=A)
    assert one >= 2 * 4 * 2 * (64 + 2) * 4 and one % 256 == 0
    assert size(prefix_len=70, prefix_pages=A, tokens=200, q_start=A, out=A + 2 ** 20) > one
    assert size(tokens=0) == 0
    assert L.s2d_cache_evict_workspace(ctypes.byref(view(kv)), ctypes.byref(evict(kv, budget=500)), ctypes.byref(n), err, 256) == 0 and n.value == 0
    assert L.s2d_cache_evict_workspace(ctypes.byref(view(kv)), ctypes.byref(evict(kv)), ctypes.byref(n), err, 256) == 0
    assert n.value >= 2 * 2 * 2 * 64 * 4
    assert L.s2d_cache_attention_workspace(ctypes.byref(view(kv)), ctypes.byref(attention(kv)), None, err, 256) == -1


def test_status_needs_a_word(kv):
    err, bits = ctypes.create_string_buffer(256), ctypes.c_int32()
    L = kv.cache_lib()
    assert L.s2d_cache_status(ctypes.byref(view(kv, status=0)), ctypes.byref(bits), None, err, 256) == -1
    assert L.s2d_cache_status(ctypes.byref(view(kv)), None, None, err, 256) == -1
    assert L.s2d_cache_status(None, ctypes.byref(bits), None, err, 256) == -1


@pytest.mark.parametrize("bad", [dict(pos=A), dict(pos=A + 4), dict(pos=A - 4), dict(q_start=A), dict(q_start=A + 4), dict(q_start=A - 8)])
def test_append_writes_lengths_over_nothing_that_it_reads(kv, bad):
    """lengths is written while other blocks still read the positions and the starts: the two entries at A here."""
    fine = dict(pos=A + 8192, q=A + 16384, k=A + 32768, v=A + 65536, q_out=A + 16384)
    assert "lengths" in refused(kv, "s2d_cache_append", view(kv), append(kv, **{**fine, **bad}))


def _rows(at, stride, row, n):
    return set().union(*(range(at + i * stride, at + i * stride + row) for i in range(n)))


def test_append_output_over_its_inputs(kv):
    """q_out's rows against those of k and v, byte by byte: every distance and pair of strides that alignment allows, rows that
    lie between each other's and rows that meet.  2 query heads and 1 KV head of 64 f16 elements: rows of 256 and 128 bytes.
    There is no device -1, so what is not refused for its rows fails before any launch."""
    L, err = kv.cache_lib(), ctypes.create_string_buffer(256)
    one = view(kv, kv_heads=1, page_stride=64 * 64, n_seq=8, lengths=A + 2 ** 20, device=-1)
    far, met, apart = A + 2 ** 22, 0, 0
    for n in (1, 2, 5):
        for out_stride in (256, 384, 512):
            for k_stride in (0, 64, 128, 256, 384, 512):
                for off in range(-1024, 1025, 64):
                    shared = bool(_rows(0, out_stride, 256, n) & _rows(off, k_stride, 128, n))
                    for name in ("k", "v"):
                        a = append(kv, tokens=n, heads=2, q=far, q_out=A + 8192, q_stride=128, q_out_stride=out_stride // 2, pos=far, past=far,
                                   **{"k": far, "v": far, name: A + 8192 + off, "k_stride": 64, "v_stride": 64, name + "_stride": k_stride // 2})
                        rc = L.s2d_cache_append(ctypes.byref(one), ctypes.byref(a), None, err, 256)
                        assert rc != 0 and (b"k or v" in err.value) == shared, (n, out_stride, k_stride, off, err.value)
                    met, apart = met + shared, apart + (not shared)
    assert met > 500 and apart > 500


def test_append_output_over_the_queries(kv):
    """The queries themselves with another stride, or rows that meet theirs, are refused; rows between theirs are not."""
    L, err = kv.cache_lib(), ctypes.create_string_buffer(256)
    v = view(kv, lengths=A + 2 ** 20, device=-1)
    for off, refuse in ((0, False), (512, False), (16, True), (496, True), (-16, True), (1024, True), (1536, False)):
        a = append(kv, q=A + 8192, q_out=A + 8192 + off, q_stride=512, q_out_stride=512, k=A + 2 ** 21, v=A + 2 ** 21, pos=A + 2 ** 21)
        L.s2d_cache_append(ctypes.byref(v), ctypes.byref(a), None, err, 256)
        assert (b"q_out" in err.value) == refuse, (off, err.value)
    assert "q_out" in refused(kv, "s2d_cache_append", v, append(kv, q_stride=512, q_out_stride=256, k=A + 2 ** 21, v=A + 2 ** 21, pos=A + 2 ** 21))


def test_attention_output_between_the_queries_rows(kv):
    """Rows of 512 bytes, 1,024 apart: out between q's rows is taken (and there is no device -1 to run it), over them refused."""
    L, err = kv.cache_lib(), ctypes.create_string_buffer(256)
    for off, refuse in ((512, False), (528, True), (496, True), (-512, False), (-496, True), (1024, True), (0, True)):
        a = attention(kv, q=A + 8192, out=A + 8192 + off, q_stride=512, out_stride=512)
        assert L.s2d_cache_attention(ctypes.byref(view(kv, device=-1)), ctypes.byref(a), None, err, 256) == (-1 if refuse else -3)
        assert (b"overlap" in err.value) == refuse, (off, err.value)
