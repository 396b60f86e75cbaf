"""The serving operators without a GPU: refusals before anything is launched, workspace queries, and the
addresses that the cache's kernels form, replayed over tables, slots and lengths they must not trust."""
import ctypes
import os
import subprocess

import pytest

from kernelcodegen_amd import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # an aligned address that is never used: every call here is refused first
OK, NULL, SHAPE, UNSUPPORTED, ARGUMENT = 0, 1, 2, 3, 5


def rows(data=P, b=0, s=128 * 8, h=128):
    return lib.Rows(data, b, s, h)


def cache(**change):
    c = dict(k=P, v=P, k_exp=P, v_exp=P, dtype=2, pages=4, page_size=16, heads=8, dim=128)
    c.update(change)
    return lib.KvCache(*[c[n] for n, _ in lib.KvCache._fields_])


def norm_rope(q=None, k=None, qo=None, ko=None, wq=P, wk=P, pos=P, freq=P, dtype=1, B=1, S=4, Hq=8, Hk=8, D=128,
              rot=128, interleaved=0, eps=1e-6):
    r = [x if x is not None else rows() for x in (q, k, qo, ko)]
    return lib.load().kcg_qk_norm_rope(*[ctypes.byref(x) for x in r], wq, wk, pos, freq, dtype, B, S, Hq, Hk, D, rot,
                                       interleaved, eps, None)


@pytest.mark.parametrize("change, status", [
    (dict(wq=None), NULL), (dict(wk=None), NULL), (dict(pos=None), NULL), (dict(freq=None), NULL),
    (dict(q=rows(None)), NULL), (dict(ko=rows(None)), NULL),
    (dict(dtype=2), ARGUMENT), (dict(dtype=-1), ARGUMENT), (dict(interleaved=2), ARGUMENT),
    (dict(eps=-1.0), ARGUMENT), (dict(eps=float("nan")), ARGUMENT), (dict(eps=float("inf")), ARGUMENT),
    (dict(S=0), SHAPE), (dict(B=0), SHAPE), (dict(Hq=0), SHAPE), (dict(Hk=-1), SHAPE), (dict(D=0), SHAPE),
    (dict(D=96), UNSUPPORTED), (dict(rot=24), UNSUPPORTED), (dict(rot=0), UNSUPPORTED), (dict(rot=144), UNSUPPORTED),
    (dict(S=1 << 21), UNSUPPORTED), (dict(S=0x7fffffff, B=0x7fffffff), UNSUPPORTED),
    (dict(q=rows(P + 1)), ARGUMENT), (dict(wq=P + 1), ARGUMENT), (dict(pos=P + 2), ARGUMENT),
    (dict(q=rows(s=-1)), ARGUMENT),
    # outputs whose rows overlap: a head's rows nearer than D, tokens nearer than their heads, broadcast
    (dict(qo=rows(h=64)), ARGUMENT), (dict(ko=rows(s=512)), ARGUMENT), (dict(qo=rows(s=0)), ARGUMENT),
    (dict(qo=rows(s=128, h=128)), ARGUMENT), (dict(qo=rows(h=1 << 60)), ARGUMENT),
])
def test_norm_rope_refusals(change, status):
    assert norm_rope(**change) == status


def test_rows_beyond_any_memory_are_refused():
    """2^48 elements times 2^16 steps do not count as none: rows of two heads would be the same."""
    far = rows(s=1 << 48, h=1 << 48)
    assert norm_rope(qo=far, S=65537, Hq=2, Hk=1) == ARGUMENT
    assert norm_rope(ko=far, S=65537, Hq=1, Hk=2) == ARGUMENT


def test_norm_rope_backward_refusals():
    L = lib.load()
    need = L.kcg_qk_norm_rope_backward_ws_bytes(1, 4, 8, 8, 128)
    assert need > 0 and need % (2 * 128 * 4) == 0
    assert L.kcg_qk_norm_rope_backward_ws_bytes(1, 0, 8, 8, 128) == 0
    assert L.kcg_qk_norm_rope_backward_ws_bytes(1, 4, 8, 8, 80) == 0

    def call(ws=P, size=need, gw=P, dq=None, gq=None):
        r = [dq or rows(), rows(), rows(), rows(), gq or rows(), rows()]
        return L.kcg_qk_norm_rope_backward(*[ctypes.byref(x) for x in r], P, P, gw, P, P, P, 1, 1, 4, 8, 8, 128, 128, 0,
                                           1e-6, ws, size, None)
    assert call(ws=None) == NULL and call(gw=None) == NULL and call(dq=rows(None)) == NULL
    assert call(size=need - 1) == ARGUMENT and call(ws=P + 4) == ARGUMENT and call(gw=P + 1) == ARGUMENT
    assert call(gq=rows(h=0)) == ARGUMENT


CACHE_REFUSALS = [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(k_exp=None), NULL), (dict(v_exp=None), NULL),
    (dict(dtype=0), ARGUMENT), (dict(dtype=7), ARGUMENT), (dict(k=P + 8), ARGUMENT), (dict(v_exp=P + 4), ARGUMENT),
    (dict(pages=0), SHAPE), (dict(heads=-8), SHAPE), (dict(page_size=0), SHAPE), (dict(dim=0), SHAPE),
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED),
    (dict(dim=96), UNSUPPORTED), (dict(pages=1 << 27), UNSUPPORTED),
]


@pytest.mark.parametrize("change, status", CACHE_REFUSALS)
def test_cache_refusals(change, status):
    L = lib.load()
    c, r = ctypes.byref(cache(**change)), ctypes.byref(rows())
    assert L.kcg_kv_cache_write(c, r, r, 1, P, 1, 4, None) == status
    assert L.kcg_kv_cache_read(c, P, r, r, 1, 1, 4, None) == status
    assert L.kcg_fmha_cache(r, c, P, 2, P, None, None, r, 1, 1, 1, 8, 1.0, None, 0, None) == status
    assert L.kcg_fmha_cache_ws_bytes(c, 2, 1, 1, 8) == 0


def test_cache_row_refusals():
    L = lib.load()
    c, r = ctypes.byref(cache()), ctypes.byref(rows())
    none, tight = ctypes.byref(rows(None)), ctypes.byref(rows(h=0))
    assert L.kcg_kv_cache_write(None, r, r, 1, P, 1, 4, None) == NULL
    assert L.kcg_kv_cache_write(c, none, r, 1, P, 1, 4, None) == NULL
    assert L.kcg_kv_cache_write(c, r, r, 1, None, 1, 4, None) == NULL
    assert L.kcg_kv_cache_write(c, r, r, 2, P, 1, 4, None) == ARGUMENT
    assert L.kcg_kv_cache_write(c, r, r, 1, P + 2, 1, 4, None) == ARGUMENT
    assert L.kcg_kv_cache_write(c, r, r, 1, P, 1, 0, None) == SHAPE
    assert L.kcg_kv_cache_write(c, r, r, 1, P, 1 << 16, 1 << 16, None) == UNSUPPORTED
    assert L.kcg_kv_cache_read(c, P, r, tight, 1, 1, 4, None) == ARGUMENT  # rows that are written must not overlap
    assert L.kcg_kv_cache_read(c, P, r, none, 1, 1, 4, None) == NULL


def test_one_memory_for_two_outputs_is_refused():
    """Which of the two rows it held in the end would be a matter of chance."""
    L = lib.load()
    assert norm_rope(qo=rows(2 * P), ko=rows(2 * P)) == ARGUMENT
    r, other = ctypes.byref(rows()), ctypes.byref(rows(2 * P))

    def backward(gq, gwq):
        return L.kcg_qk_norm_rope_backward(r, r, r, r, gq, r, P, P, gwq, P, P, P, 1, 1, 4, 8, 8, 128, 128, 0, 1e-6, P,
                                           1 << 30, None)
    assert backward(r, 2 * P) == ARGUMENT and backward(other, P) == ARGUMENT
    assert L.kcg_kv_cache_read(ctypes.byref(cache()), P, other, other, 1, 1, 4, None) == ARGUMENT


@pytest.mark.parametrize("change, status", [
    (dict(table=None), NULL), (dict(context=None), NULL), (dict(q=rows(None)), NULL), (dict(out=rows(None)), NULL),
    (dict(o_dtype=2), ARGUMENT), (dict(scale=float("nan")), ARGUMENT), (dict(scale=float("inf")), ARGUMENT),
    (dict(table=P + 1), ARGUMENT), (dict(drafts=P + 2), ARGUMENT), (dict(tree=P + 4), ARGUMENT),
    (dict(ws=P + 8, size=1 << 20), ARGUMENT), (dict(ws=P, size=-1), ARGUMENT), (dict(out=rows(h=1)), ARGUMENT),
    (dict(N=0), SHAPE), (dict(B=-1), SHAPE), (dict(width=0), SHAPE), (dict(Hq=0), SHAPE),
    (dict(N=65), UNSUPPORTED), (dict(Hq=12), UNSUPPORTED), (dict(width=1 << 28), UNSUPPORTED),
    (dict(B=1 << 24, width=1 << 10), UNSUPPORTED),
])
def test_fmha_cache_refusals(change, status):
    a = dict(q=rows(), table=P, width=4, context=P, drafts=None, tree=None, out=rows(), o_dtype=1, B=1, N=1, Hq=8,
             scale=1.0, ws=None, size=0)
    a.update(change)
    got = lib.load().kcg_fmha_cache(ctypes.byref(a["q"]), ctypes.byref(cache()), a["table"], a["width"], a["context"],
                                    a["drafts"], a["tree"], ctypes.byref(a["out"]), a["o_dtype"], a["B"], a["N"],
                                    a["Hq"], a["scale"], a["ws"], a["size"], None)
    assert got == status


@pytest.mark.parametrize("B, page", [(64, 256), (33, 256), (64, 128), (1024, 64)])
def test_fmha_cache_refuses_tables_whose_chunks_do_not_count_in_32_bits(B, page):
    """Units are counted in 32 bits on the device, over whatever lengths it finds: the tables' room bounds them."""
    L, width = lib.load(), (1 << 35) // page // B
    c, r = cache(page_size=page), rows()

    def call(width):
        return L.kcg_fmha_cache(ctypes.byref(r), ctypes.byref(c), P, width, P, None, None, ctypes.byref(rows(h=1)), 1, B,
                                1, 8, 1.0, None, 0, None)
    # (the output's rows overlap, so that nothing is launched for what is accepted)
    assert call(width) == ARGUMENT and L.kcg_fmha_cache_ws_bytes(ctypes.byref(c), width, B, 1, 8) > 0
    assert call(width + 1) == UNSUPPORTED and L.kcg_fmha_cache_ws_bytes(ctypes.byref(c), width + 1, B, 1, 8) == 0


def test_extents_beyond_32_bits_are_refused():
    """The C interface counts tokens and pages in 32 bits: 2^32 + 4 of them must not become 4."""
    torch = pytest.importorskip("torch")
    from kernelcodegen_amd import ops
    many = (1 << 32) + 4
    # tensors without memory, whose device index is that of the cache
    handle = ops.KvCache.__new__(ops.KvCache)
    handle.index, handle.heads, handle.dim, handle._c = -1, 8, 128, cache(k=None)
    rows = torch.empty(1, 8, 128, dtype=torch.bfloat16, device="meta").expand(many, 8, 128)
    slots = torch.empty(many, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.kv_cache_write(handle, rows, rows, slots)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.kv_cache_read(handle, slots, out=(rows, rows))
    q = torch.empty(1, 1, 8, 128, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.fmha_cache(q, handle, slots.view(1, many), torch.empty(1, dtype=torch.int32, device="meta"), out=q)


def test_cache_addresses_stay_inside(tmp_path):
    """tests/kv_cache_index_model.cc replays csrc/kv_cache_index.h on the host."""
    exe = str(tmp_path / "model")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "kernelcodegen_amd", "csrc"),
                    os.path.join(ROOT, "tests", "kv_cache_index_model.cc"), "-o", exe], check=True)
    out = subprocess.run([exe], stdout=subprocess.PIPE, text=True, timeout=120)
    assert out.returncode == 0, out.stdout
    assert "all inside" in out.stdout
