"""CPU: argument checks of the paged K/V cache's C entry points and wrappers, before any device is touched."""
import ctypes as C

import pytest
import torch

from pika_h3_flex_b200 import _lib

BUF = (C.c_char * 8192)()
BASE = (C.addressof(BUF) + 255) & ~255


def good():
    p = _lib.CacheAttnParams()
    c, b = p.cache, p.batch
    c.k = c.v = BASE
    for x in ("k", "v"):
        setattr(c, f"{x}_stride_page", 16 * 128)
        setattr(c, f"{x}_stride_token", 128)
        setattr(c, f"{x}_stride_head", 128)
    c.n_pages, c.page_size, c.heads, c.d = 4, 16, 1, 128
    b.pages = b.lengths = b.starts = BASE
    b.pages_stride, b.n_seqs, b.max_pages, b.rows = 4, 1, 4, 1
    p.q, p.o = BASE, BASE + 4096
    p.q_stride_l = p.q_stride_h = p.o_stride_l = p.o_stride_h = 128
    p.heads, p.causal = 1, 1
    p.workspace, p.workspace_bytes = BASE, 1
    return p


def set_in(path, value):
    def f(p):
        *outer, last = path.split(".")
        for x in outer:
            p = getattr(p, x)
        setattr(p, last, value)
    return f


BAD = [
    ("cache.k", None, "ARG"), ("cache.v", None, "ARG"), ("batch.pages", None, "ARG"), ("batch.lengths", None, "ARG"), ("batch.starts", None, "ARG"),
    ("cache.quantised", 2, "ARG"), ("cache.quantised", 1, "ARG"), ("cache.k_exp", BASE, "ARG"), ("batch.pages_stride", -1, "ARG"),
    ("cache.d", 64, "SHAPE"), ("cache.n_pages", 0, "SHAPE"), ("cache.heads", 0, "SHAPE"), ("cache.page_size", 24, "SHAPE"), ("cache.page_size", 0, "SHAPE"),
    ("cache.page_size", 65552, "SHAPE"), ("batch.n_seqs", 0, "SHAPE"), ("batch.max_pages", 0, "SHAPE"), ("batch.max_pages", 1 << 25, "SHAPE"),
    ("batch.rows", 0, "SHAPE"), ("batch.rows", 1 << 30, "SHAPE"),
    ("cache.k", BASE + 2, "ALIGN"), ("cache.v_stride_token", 100, "ALIGN"), ("cache.k_stride_head", 0, "ALIGN"), ("cache.v_stride_page", -128, "ALIGN"),
]
BAD_ATTN = [("q", None, "ARG"), ("o", None, "ARG"), ("o", BASE, "ARG"), ("causal", 2, "ARG"), ("max_new", -1, "ARG"), ("heads", 0, "SHAPE"), ("q", BASE + 8, "ALIGN"), ("o_stride_h", 0, "ALIGN"),
            ("q_stride_l", -128, "ALIGN"), ("q_stride_h", 0, "ALIGN"), ("o_stride_l", 4, "ALIGN")]


@pytest.mark.parametrize("path,value,code", BAD + BAD_ATTN)
def test_attention_refuses(lib, path, value, code):
    p = good()
    set_in(path, value)(p)
    assert lib.h3a_cache_attn(C.byref(p), None) == getattr(_lib, "H3A_ERR_" + code)


@pytest.mark.parametrize("path,value,code", BAD)
def test_write_and_read_refuse(lib, path, value, code):
    p = good()
    set_in(path, value)(p)
    for f in (lib.h3a_cache_write, lib.h3a_cache_read):
        assert f(C.byref(p.cache), C.byref(p.batch), BASE, 128, 128, BASE, 128, 128, None, None) == getattr(_lib, "H3A_ERR_" + code)


def test_packed_rows_are_checked(lib):
    p = good()
    c, b = C.byref(p.cache), C.byref(p.batch)
    for f in (lib.h3a_cache_write, lib.h3a_cache_read):
        assert f(None, b, BASE, 128, 128, BASE, 128, 128, None, None) == _lib.H3A_ERR_ARG
        assert f(c, None, BASE, 128, 128, BASE, 128, 128, None, None) == _lib.H3A_ERR_ARG
        assert f(c, b, None, 128, 128, BASE, 128, 128, None, None) == _lib.H3A_ERR_ARG
        assert f(c, b, BASE, 128, 100, BASE, 128, 128, None, None) == _lib.H3A_ERR_ALIGN
        assert f(c, b, BASE, 128, 128, BASE + 4, 128, 128, None, None) == _lib.H3A_ERR_ALIGN
    assert lib.h3a_cache_read(c, b, BASE, 0, 128, BASE, 128, 128, None, None) == _lib.H3A_ERR_ALIGN  # a written row must not repeat


def test_heads_must_divide(lib):
    p = good()
    p.cache.heads, p.heads = 2, 3
    assert lib.h3a_cache_attn(C.byref(p), None) == _lib.H3A_ERR_SHAPE
    assert lib.h3a_cache_attn(None, None) == _lib.H3A_ERR_ARG
    need = C.c_size_t(0)
    assert lib.h3a_cache_attn_workspace_bytes(C.byref(p), C.byref(need)) == _lib.H3A_ERR_SHAPE
    assert lib.h3a_cache_attn_workspace_bytes(None, C.byref(need)) == _lib.H3A_ERR_ARG


def test_struct_sizes_match_a_c_compiler(tmp_path):
    import os
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include "h3attn.h"\nint main(void) { printf("%zu %zu %zu\\n", sizeof(h3a_cache), sizeof(h3a_cache_batch), '
                   'sizeof(h3a_cache_attn_params)); return 0; }\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [C.sizeof(_lib.Cache), C.sizeof(_lib.CacheBatch), C.sizeof(_lib.CacheAttnParams)]


def test_wrappers_refuse_cpu_tensors(lib):
    import pika_h3_flex_b200 as h3

    pool = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        h3.KVCache(pool, pool)
    with pytest.raises(RuntimeError, match="no CPU path"):
        h3.CacheBatch(i32[None], i32, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        h3.cache_attn(pool[0], None, None)


@pytest.mark.parametrize("which", ["k_exp", "v_exp"])
@pytest.mark.parametrize("dim", ["page", "token", "head"])
def test_exponents_of_a_written_cache_must_not_repeat(lib, which, dim):
    """A byte that several rows share cannot take all their exponents; what is only read may repeat, but not run backwards."""
    def quantised(stride):
        p = good()
        c = p.cache
        c.quantised, c.k_exp, c.v_exp = 1, BASE, BASE + 1024
        for x in ("k", "v"):
            for d, n in (("page", 16 * 128), ("token", 128), ("head", 128)):
                setattr(c, f"{x}_exp_stride_{d}", n // 128)
        setattr(c, f"{which}_stride_{dim}", stride)
        return p

    def calls(p):  # none of them gets as far as a launch: what comes after the cache's checks is refused too
        p.heads = 0
        c, b = C.byref(p.cache), C.byref(p.batch)
        return (lib.h3a_cache_write(c, b, None, 128, 128, BASE, 128, 128, None, None),
                lib.h3a_cache_read(c, b, None, 128, 128, BASE, 128, 128, None, None), lib.h3a_cache_attn(C.byref(p), None))

    bad, arg, shape = _lib.H3A_ERR_ALIGN, _lib.H3A_ERR_ARG, _lib.H3A_ERR_SHAPE
    assert calls(quantised(0)) == (bad, arg, shape)
    assert calls(quantised(-1)) == (bad, bad, bad)
    assert calls(quantised(1)) == (arg, arg, shape)


def test_a_workspace_has_to_have_its_bytes():
    """An expanded tensor counts more bytes than it has, and a strided one has gaps."""
    from pika_h3_flex_b200 import cache

    cpu = torch.device("cpu")
    cache._check_workspace(torch.empty(1 << 20, dtype=torch.uint8), cpu)
    for w in (torch.empty(1, dtype=torch.uint8).expand(1 << 20), torch.empty(64, 64, dtype=torch.uint8)[:, ::2], torch.empty(64, 64)[:, :32]):
        with pytest.raises(ValueError, match="contiguous"):
            cache._check_workspace(w, cpu)
    with pytest.raises(ValueError, match="workspace on cpu"):
        cache._check_workspace(torch.empty(64, dtype=torch.uint8), torch.device("cuda:0"))
