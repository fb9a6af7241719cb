"""The paged cache's argument checks, through the C ABI and the tensor-level wrappers, without a GPU."""
import ctypes as C

import pytest
import torch


def _pool(L, **kw):
    p = L.PagedPool()
    p.k_pages = p.v_pages = p.k_scale = p.v_scale = p.k_bounds = 4096
    p.num_pages, p.num_kv_heads, p.page_size, p.head_dim, p.dtype, p.format = 10, 2, 64, 128, L.BF16, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(head_dim=96), "ERR_UNSUPPORTED"), (dict(page_size=48), "ERR_UNSUPPORTED"), (dict(page_size=256), "ERR_UNSUPPORTED"),
    (dict(format=3), "ERR_INVALID_ARG"), (dict(dtype=2), "ERR_INVALID_ARG"), (dict(num_pages=0), "ERR_INVALID_ARG"),
    (dict(num_kv_heads=0), "ERR_INVALID_ARG"), (dict(k_pages=None), "ERR_INVALID_ARG"), (dict(v_scale=None), "ERR_INVALID_ARG"),
    (dict(v_pages=4100), "ERR_INVALID_ARG"), (dict(num_pages=2 ** 30, num_kv_heads=4), "ERR_INVALID_ARG"),
])
def test_pools_that_are_refused(change, code):
    from longcontext_sqattn_paddle_b200 import _lib as L
    p = _pool(L, **change)
    t = L.Tensor(4096, 1024, 128, 256)
    args = (C.addressof(t), C.addressof(t), 1, 5, 4096, 4, 4, 4096, None, None)
    assert L.lib.sqattn_paged_write(C.addressof(p), *args) == getattr(L, code)
    assert L.lib.sqattn_paged_read(C.addressof(p), *args) == getattr(L, code)
    d = L.PagedDecodeArgs(pool=C.addressof(p), batch=1, num_q_heads=4, max_pages=4, block_table=4096, kv_lens=4096, table_stride=4)
    assert L.lib.sqattn_paged_decode_workspace_bytes(C.byref(d)) == 0
    assert L.lib.sqattn_paged_decode(C.byref(d), None) == getattr(L, code)
    s = L.PagedSelectArgs(pool=C.addressof(p), batch=1, num_q_heads=4, max_pages=4, block_table=4096, kv_lens=4096, table_stride=4, budget=2)
    assert L.lib.sqattn_paged_select_workspace_bytes(C.byref(s)) == 0
    assert L.lib.sqattn_paged_select(C.byref(s), None) == getattr(L, code)


def test_rows_and_tables_that_are_refused():
    from longcontext_sqattn_paddle_b200 import _lib as L
    p = _pool(L)
    t, odd = L.Tensor(4096, 1024, 128, 256), L.Tensor(4096, 1024, 128, 250)

    def call(k=t, v=t, batch=1, rows=5, table=4096, max_pages=4, positions=4096, pool=C.addressof(p)):
        a = (pool, C.addressof(k), C.addressof(v), batch, rows, table, 4, max_pages, positions, None, None)
        return {L.lib.sqattn_paged_write(*a), L.lib.sqattn_paged_read(*a)}

    for kw in (dict(k=odd), dict(v=odd), dict(k=L.Tensor(4104, 1024, 128, 256)), dict(batch=0), dict(batch=70000), dict(rows=0),
               dict(table=None), dict(max_pages=0), dict(positions=None), dict(pool=None), dict(k=L.Tensor(None, 1024, 128, 256))):
        assert call(**kw) == {L.ERR_INVALID_ARG}, kw


def test_attention_and_selection_that_are_refused():
    from longcontext_sqattn_paddle_b200 import _lib as L
    p = _pool(L)

    def decode(**kw):
        a = L.PagedDecodeArgs(pool=C.addressof(p), batch=1, num_q_heads=4, max_pages=4, block_table=4096, kv_lens=4096, table_stride=4)
        a.q.ptr = a.o.ptr = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return L.lib.sqattn_paged_decode(C.byref(a), None)

    assert decode(num_q_heads=34) == L.ERR_UNSUPPORTED                   # 17 query heads per KV head
    for kw in (dict(num_q_heads=3), dict(num_q_heads=0), dict(kv_lens=None), dict(o_dtype=5), dict(max_kv_len=-1), dict(pages=4096),
               dict(sm_scale=float("nan")), dict(sm_scale=-1.0), dict(sm_scale=float("inf")), dict(block_table=None), dict(pool=None)):
        assert decode(**kw) == L.ERR_INVALID_ARG, kw
    a = L.PagedDecodeArgs(pool=C.addressof(p), batch=1, num_q_heads=4, max_pages=4, block_table=4096, kv_lens=4096, table_stride=4)
    assert L.lib.sqattn_paged_decode(C.byref(a), None) == L.ERR_INVALID_ARG and b"null" in L.lib.sqattn_last_error_string()

    def select(**kw):
        a = L.PagedSelectArgs(pool=C.addressof(p), batch=1, num_q_heads=4, max_pages=4, block_table=4096, kv_lens=4096, table_stride=4,
                              budget=4, sink_pages=1, recent_pages=1, out=4096)
        a.q.ptr = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return L.lib.sqattn_paged_select(C.byref(a), None)

    assert select(max_pages=131073) == L.ERR_UNSUPPORTED
    for kw in (dict(budget=0), dict(sink_pages=-1), dict(recent_pages=-1), dict(sink_pages=3, recent_pages=2),
               dict(sink_pages=2 ** 31 - 1, recent_pages=2 ** 31 - 1), dict(num_q_heads=5), dict(out=None), dict(kv_lens=None)):
        assert select(**kw) == L.ERR_INVALID_ARG, kw
    assert select() == L.ERR_WORKSPACE
    p.k_bounds = None
    assert select() == L.ERR_INVALID_ARG and b"bounds" in L.lib.sqattn_last_error_string()


def test_tensors_that_are_refused():
    """Shapes and types are checked before the device: no tensor below is on a GPU."""
    from longcontext_sqattn_paddle_b200 import ops
    z = torch.zeros
    pages, scale = z(3, 2, 16, 64, dtype=torch.int8), z(3, 2, 16)
    for args in ((pages, pages), (pages, pages, scale), (pages, pages, scale, scale.half()), (pages, z(3, 2, 16, 64), scale, scale),
                 (z(3, 2, 24, 64, dtype=torch.int8),) * 2 + (z(3, 2, 24),) * 2, (z(3, 2, 16, 80, dtype=torch.int8),) * 2 + (scale, scale),
                 (pages, pages, scale, scale, z(3, 2, 2, 128).half()), (z(3, 2, 16, 64).half(),) * 2 + (scale, scale)):
        with pytest.raises(ValueError):
            ops.PagedPool(*args, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.PagedPool(z(3, 2, 16, 64).half(), z(3, 2, 16, 64).half(), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.PagedPool(z(3, 2, 16, 64), z(3, 2, 16, 64))
    with pytest.raises(ValueError):
        ops.PagedPool.allocate(3, 16, 2, 64, kv_format="int2")
    with pytest.raises(RuntimeError):
        ops.PagedPool(pages, pages, scale, scale, dtype=torch.float16)   # all well, but no CUDA tensors


def test_page_bookkeeping():
    from longcontext_sqattn_paddle_b200.cache_hub import PageAllocator
    a = PageAllocator(num_pages=10, page_size=16, batch_size=3, max_pages=6)
    assert a.reserve(0, 1) == [0] and a.reserve(0, 16) == [] and a.reserve(0, 17) == [1]
    assert a.reserve(1, 96) == [2, 3, 4, 5, 6, 7] and a.reserve(2, 0) == []
    with pytest.raises(ValueError):
        a.reserve(0, 97)
    with pytest.raises(RuntimeError):
        a.reserve(2, 33)
    assert a.pages[2] == [] and len(a.free) == 2              # a refused reservation takes nothing
    assert a.release(1) == 6 and a.release(1) == 0
    assert sorted(a.reserve(2, 90)) == [2, 3, 4, 5, 6, 7] and sorted(a.free + a.pages[0] + a.pages[2]) == list(range(10))


def test_selection_budgets_that_are_refused():
    from longcontext_sqattn_paddle_b200.cache_hub import PagedKVCache
    with pytest.raises(ValueError):
        PagedKVCache(0, 1, 1, 64, 2, 4, 64, torch.float16, select_pages=2, sink_pages=1, recent_pages=2, device="cpu")


def test_import_without_the_inductor_allocator():
    """A torch build without that private module has the public allocator."""
    import os
    import subprocess
    import sys
    code = ("import torch\ndel torch._C._dynamo.guards\nfrom longcontext_sqattn_paddle_b200 import ops\n"
            "assert ops._empty_strided is None\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr
