"""The paged cache's and the packed attention's C entries without a GPU: their structures, what
they refuse, and that there is no CPU path."""
import ctypes
import re

import pytest
import torch

EINVAL, EALIGN, EUNSUPPORTED = -1, -2, -3


@pytest.mark.parametrize("name,cls,layout", [
    ("srdit_kv_pages", "KvPages", "KV_PAGES_LAYOUT"),
    ("srdit_seq_attn_args", "SeqAttnArgs", "SEQ_ATTN_LAYOUT")])
def test_structs_match_the_header(srdit, name, cls, layout):
    lib = srdit._lib
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), lib.HEADER.read_text(),
                     re.S).group(1)
    names = re.findall(r"(\w+)(?:\[\d\])?\s*[,;]", body)
    fields = getattr(lib, cls)._fields_
    assert names == [f[0] for f in fields]
    # the packed layout puts the n-th value into the n-th field
    a, st = getattr(lib, cls)(), getattr(lib, layout)
    width = [f[1]._length_ if hasattr(f[1], "_length_") else 1 for f in fields]
    st.pack_into(a, 0, *range(1, sum(width) + 1))
    at = 1
    for (f, _), w in zip(fields, width):
        got = getattr(a, f)
        assert (list(got) if w > 1 else got) == (list(range(at, at + w)) if w > 1 else at), f
        at += w


def _pages(lib, **kw):
    v = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, code=0, dtype=0, pages=9,
             page_size=16, Hkv=2, D=64, k_stride=(2048, 128, 64), v_stride=(2048, 128, 64),
             ks_stride=(32, 2, 1), vs_stride=(32, 1, 16), table=5 << 20, table_stride=4,
             table_width=4, B=3)
    v.update(kw)
    return _fill(lib.KvPages(), v)


def _fill(a, v):
    for name, x in v.items():
        if isinstance(x, tuple):
            getattr(a, name)[:] = x
        else:
            setattr(a, name, x)
    return a


PAGES = [
    (dict(B=-1), EINVAL), (dict(pages=-1), EINVAL), (dict(Hkv=0), EINVAL), (dict(D=0), EINVAL),
    (dict(page_size=0), EINVAL), (dict(table_width=-1), EINVAL), (dict(dtype=2), EINVAL),
    (dict(code=2), EINVAL), (dict(k=None), EINVAL), (dict(v_scale=None), EINVAL),
    (dict(table=None), EINVAL), (dict(D=136), EUNSUPPORTED), (dict(D=72), EUNSUPPORTED),
    (dict(code=-1, D=60), EUNSUPPORTED), (dict(page_size=8), EUNSUPPORTED),
    (dict(page_size=48), EUNSUPPORTED), (dict(page_size=192), EUNSUPPORTED),
    (dict(Hkv=1025), EUNSUPPORTED), (dict(table_width=1 << 28), EUNSUPPORTED),
    (dict(k=(1 << 20) + 8), EALIGN), (dict(v_stride=(2048, 120, 64)), EALIGN),
    (dict(table=(5 << 20) + 2), EALIGN), (dict(k_scale=(3 << 20) + 2), EALIGN),
    (dict(k_stride=(2048, 0, 64)), EINVAL), (dict(v_stride=(-2048, 128, 64)), EINVAL),
    (dict(ks_stride=(32, 2, 0)), EINVAL)]


def _rows_call(lib, write, pages=None, **kw):
    v = dict(k=6 << 20, k_stride=(128, 64), v=7 << 20, v_stride=(128, 64), T=5, cu=8 << 20,
             lens=9 << 20)
    v.update(kw)
    p = _pages(lib, **(pages or {}))
    st = [(ctypes.c_longlong * 2)(*v[x]) if v[x] else None for x in ("k_stride", "v_stride")]
    args = [ctypes.byref(p), v["k"], st[0], v["v"], st[1], v["T"], v["cu"]]
    if write:
        return lib.lib().srdit_kv_write(*args, v["lens"], None)
    return lib.lib().srdit_kv_read(*args, None)


@pytest.mark.parametrize("write", (True, False))
@pytest.mark.parametrize("pages,rc", PAGES)
def test_page_refusals(srdit, write, pages, rc):
    assert _rows_call(srdit._lib, write, pages) == rc


@pytest.mark.parametrize("write", (True, False))
@pytest.mark.parametrize("kw,rc", [
    (dict(T=0), 0), (dict(T=-1), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL),
    (dict(k_stride=None), EINVAL), (dict(cu=None), EINVAL), (dict(k=(6 << 20) + 8), EALIGN),
    (dict(v_stride=(128, 60)), EALIGN), (dict(cu=2), EALIGN)])
def test_row_refusals(srdit, write, kw, rc):
    assert _rows_call(srdit._lib, write, **kw) == rc


def test_read_and_write_differ(srdit):
    lib = srdit._lib
    assert _rows_call(lib, True, lens=None) == EINVAL
    assert _rows_call(lib, True, lens=3) == EALIGN
    assert _rows_call(lib, False, k_stride=(0, 64)) == EINVAL   # two tokens in one place
    assert _rows_call(lib, True, pages=dict(B=0)) == 0
    assert lib.lib().srdit_kv_write(None, *[None] * 4, 5, None, None, None) == EINVAL


def _attn(lib, pages=None, workspace=False, **kw):
    v = dict(q=10 << 20, k=11 << 20, v=12 << 20, out=13 << 20, dtype=0, T=6, Tk=6, B=3, H=4, Hkv=2,
             D=64, q_stride=(256, 64), k_stride=(128, 64), v_stride=(128, 64), o_stride=(256, 64),
             cu_q=14 << 20, kv_lens=15 << 20, max_q=2, scale=0.125)
    v.update(kw)
    a = _fill(lib.SeqAttnArgs(), v)
    if pages is not None:
        p = _pages(lib, **pages)
        a.pages = ctypes.addressof(p)
    if workspace:
        return lib.lib().srdit_seq_attn_workspace(ctypes.byref(a))
    return lib.lib().srdit_seq_attn(ctypes.byref(a), None)


@pytest.mark.parametrize("pages", (None, {}))
@pytest.mark.parametrize("kw,rc", [
    (dict(T=0), 0), (dict(H=0), 0), (dict(T=-1), EINVAL), (dict(Hkv=0), EINVAL),
    (dict(H=3), EINVAL), (dict(dtype=2), EINVAL), (dict(max_q=-1), EINVAL),
    (dict(max_kv=-1), EINVAL), (dict(q=None), EINVAL), (dict(out=None), EINVAL),
    (dict(scale=0.0), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL),
    (dict(cu_q=None, T=7), EINVAL), (dict(q=(10 << 20) + 8), EALIGN), (dict(cu_q=2), EALIGN),
    (dict(q_stride=(256, 60)), EALIGN), (dict(o_stride=(256, 0)), EINVAL),
    (dict(q_stride=(0, 64)), EINVAL), (dict(q_stride=(256, 0)), EINVAL),
    (dict(q_stride=(-256, 64)), EALIGN),
    (dict(T=1 << 25), EUNSUPPORTED)])
def test_attention_refusals(srdit, pages, kw, rc):
    assert _attn(srdit._lib, pages, **kw) == rc
    assert _attn(srdit._lib, pages, workspace=True, **kw) == 0


@pytest.mark.parametrize("pages,rc", PAGES)
def test_attention_page_refusals(srdit, pages, rc):
    assert _attn(srdit._lib, pages) == rc


@pytest.mark.parametrize("pages,kw,rc", [
    (dict(Hkv=1), {}, EINVAL), (dict(B=2), {}, EINVAL), (dict(D=32), {}, EINVAL),
    (dict(dtype=1), {}, EINVAL), ({}, dict(kv_lens=None), EINVAL), ({}, dict(kv_lens=2), EALIGN),
    (None, dict(k=None), EINVAL), (None, dict(v=None), EINVAL), (None, dict(Tk=-1), EINVAL),
    (None, dict(D=60), EUNSUPPORTED), (None, dict(D=136), EUNSUPPORTED),
    (None, dict(k_stride=(128, 60)), EALIGN), (None, dict(v_stride=(0, 64)), EINVAL),
    (None, dict(cu_k=2), EALIGN), (None, dict(cu_q=None, Tk=7), EINVAL),
    (None, dict(cu_k=16 << 20, Tk=2 ** 31 - 255), EUNSUPPORTED)])
def test_attention_key_refusals(srdit, pages, kw, rc):
    assert _attn(srdit._lib, pages, **kw) == rc


def test_no_cpu_path(srdit):
    err, ops = srdit._lib.SrditError, srdit.ops
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    pool = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: ops.kv_write(x, x, pool, pool, i, i[:, 0]),
                 lambda: ops.kv_read(pool, pool, i, i[:, 0], total=2),
                 lambda: ops.paged_attn(x, pool, pool, i, i[:, 0]),
                 lambda: ops.packed_attn(x, x, x, i[:, 0])):
        with pytest.raises(err):
            call()


# ------------------------------------------------------------------ the kernels' sources
from tests.test_bounded_waits_cpu import _code, _without_single_threads  # noqa: E402


@pytest.mark.parametrize("name", ("seq_step.cu", "seq_chunk.cu"))
def test_a_warp_gives_up_as_one(name):
    """As tests/test_bounded_waits_cpu.py has it for the other kernels: a wait of a whole warp
    has one answer, or none is asked for and the abort flag is voted on."""
    text = _code(name)
    assert "mbar_wait" in text and "named_barrier" not in text
    shared = _without_single_threads(text)
    for m in re.finditer(r"\bmbar_wait\(", shared):
        assert re.search(r"[;{}]\s*$", shared[:m.start()]), shared[m.start() - 40:m.end() + 60]
        assert shared[m.start():shared.index(";", m.end())].endswith("abort_flag)")
        assert "if (__any_sync(0xffffffffu, *abort_flag != 0u)) break;" in shared


def test_clusters_are_never_launched_programmatically(srdit):
    text = (srdit._lib.PKG / "csrc" / "seq_step.cu").read_text()
    body = re.search(r"^static int launch\(.*?^\}", text, re.S | re.M).group(0)
    assert "launch_clusters(" in body and "SRDIT_LAUNCH" not in body
    assert text.count("step_kernel<T, DP, NT, CODE>") == 2   # its shared memory, its launch


# ------------------------------------------------------------------ how a call is run
STEP, STEP_SHARES, CHUNK, CHUNK_SHARES, CHUNK_REST = 1, 2, 3, 4, 5


def _way(lib, pages, B, T, H, Hkv, kv=0, max_q=0, causal=1, D=128, Tk=0, width=None, code=-1):
    v = dict(q=10 << 20, k=11 << 20, v=12 << 20, out=13 << 20, T=T, Tk=Tk, B=B, H=H, Hkv=Hkv, D=D,
             q_stride=(H * D, D), k_stride=(Hkv * D, D), v_stride=(Hkv * D, D), o_stride=(H * D, D),
             cu_q=14 << 20, kv_lens=15 << 20, max_q=max_q, max_kv=kv, causal=causal, scale=0.125)
    a = _fill(lib.SeqAttnArgs(), v)
    if pages:
        st = (16 * Hkv * D, Hkv * D, D)
        p = _pages(lib, B=B, Hkv=Hkv, D=D, code=code, k_stride=st, v_stride=st,
                   ks_stride=(16 * Hkv, Hkv, 1), vs_stride=(16 * Hkv, Hkv, 1),
                   table_width=width or max(1, -(-kv // 16)))
        a.pages = ctypes.addressof(p)
    L = lib.lib()
    ws = L.srdit_seq_attn_workspace(ctypes.byref(a))
    way = L.srdit_seq_attn_way(ctypes.byref(a))
    # parts of rows meet in the workspace (parts of clusters only where they are more than 8)
    assert way == STEP or (ws > 0) == (way in (STEP_SHARES, CHUNK_SHARES, CHUNK_REST))
    return way


@pytest.mark.parametrize("kw,way", [
    (dict(B=4, T=4, H=32, Hkv=8, kv=1024, max_q=1), STEP),
    (dict(B=32, T=32, H=32, Hkv=8, kv=4096, max_q=1), STEP_SHARES),
    (dict(B=1100, T=1100, H=32, Hkv=8, kv=4096, max_q=1), STEP),           # more than are kept
    (dict(B=32, T=32, H=32, Hkv=8, kv=4096, max_q=1, code=1), STEP_SHARES),
    (dict(B=8, T=32, H=16, Hkv=4, kv=64, max_q=4), STEP),                  # 16 rows a key head
    (dict(B=8, T=40, H=16, Hkv=4, kv=64, max_q=5), CHUNK),
    (dict(B=1, T=64, H=32, Hkv=8, kv=32768), CHUNK_SHARES),
    (dict(B=1, T=64, H=32, Hkv=8, kv=300), CHUNK),
    (dict(B=1, T=6912, H=24, Hkv=24, kv=13824, causal=0), CHUNK_REST),
    (dict(B=1, T=6912, H=24, Hkv=24, kv=512, causal=0), CHUNK),
    (dict(B=500, T=6912, H=24, Hkv=24, kv=13824, causal=0), CHUNK),        # more pieces than are kept
    (dict(B=1, T=1400, H=32, Hkv=8, kv=1 << 20), CHUNK_SHARES),
    (dict(B=1, T=1400, H=32, Hkv=8, kv=1 << 20, width=1 << 26), CHUNK),    # key tiles beyond 32 bits
])
def test_ways_over_pages(srdit, kw, way):
    assert _way(srdit._lib, True, **kw) == way


@pytest.mark.parametrize("kw,way", [
    (dict(B=1, T=1, H=1, Hkv=1, Tk=1), CHUNK), (dict(B=16, T=4000, H=24, Hkv=24, Tk=4000), CHUNK),
    (dict(B=1, T=8192, H=32, Hkv=8, Tk=8192), CHUNK),
    (dict(B=1, T=300, H=4, Hkv=4, Tk=20000), CHUNK_SHARES),
    (dict(B=1, T=2304, H=24, Hkv=24, Tk=6912, causal=0), CHUNK_REST)])
def test_ways_of_packed_rows(srdit, kw, way):
    assert _way(srdit._lib, False, **kw) == way


def test_the_extension_leaves_what_it_does_not_know(srdit):
    """Without CUDA tensors it takes nothing: the wrappers say what is wrong."""
    ext = srdit._lib.calls()
    assert ext is not None
    x, i = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 1, dtype=torch.int32)
    pool = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    assert ext.kv_write(x, x, pool, pool, i, i[:, 0], None, None, None) is None
    assert ext.kv_read(pool, pool, i, i[:, 0], x, x, None, None) is None
    assert ext.paged_attn(x, pool, pool, i, i[:, 0], x, None, 1, 1, True, None, None, None,
                          None) is None
    assert ext.packed_attn(x, x, x, i[:, 0], x, None, True, None, None) is None
    for f, n in ((ext.kv_write, 9), (ext.kv_read, 8), (ext.paged_attn, 14), (ext.packed_attn, 9)):
        assert f() is None and f(*[None] * n) is None and f(*[3] * n) is None
    with pytest.raises(TypeError):
        ext.init(1)
