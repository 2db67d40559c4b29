"""The paged fp8 cache without a GPU: what the C ABI and the package refuse before anything is launched, and the
oracle against hand-made values."""
import ctypes
import os
import re

import pytest
import torch

from cutlass_flash_atten_fp8_b200 import PagedKVCache, _lib, flash_attention_paged_kv, paged_kv_append, paged_kv_read
from cutlass_flash_atten_fp8_b200.build import LIB_PATH, REPO_DIR
from oracle import paged_kv_oracle as po

FAKE = 0x10000                       # never dereferenced: validation fails first


def cache_params(**kw):
    p = dict(k=FAKE, v=FAKE, k_descale=FAKE, v_descale=FAKE, num_pages=8, heads_kv=2, page_size=16, head_dim=64, fp8_format=0,
             batch=2, page_table=FAKE, table_width=4, table_stride=4, seqlens=FAKE, cu_seqlens=None, tokens=2, status_word=FAKE)
    p.update(kw)
    return _lib.Fa8KvCache(**p)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_descale=None), dict(v_descale=None), dict(page_table=None), dict(seqlens=None),
              dict(num_pages=0), dict(heads_kv=0), dict(heads_kv=-1), dict(batch=0), dict(table_width=0), dict(tokens=-1),
              dict(table_stride=3), dict(fp8_format=2), dict(k=FAKE + 8), dict(v=FAKE + 4), dict(k_descale=FAKE + 2),
              dict(v_descale=FAKE + 1), dict(page_table=FAKE + 2), dict(seqlens=FAKE + 1), dict(cu_seqlens=FAKE + 2),
              dict(status_word=FAKE + 3), dict(tokens=3)]
UNSUPPORTED_CACHES = [dict(head_dim=0), dict(head_dim=48), dict(head_dim=288), dict(page_size=8), dict(page_size=24), dict(page_size=256),
                      dict(page_size=0), dict(table_width=1 << 27, table_stride=1 << 27, page_size=16), dict(num_pages=1 << 30, heads_kv=2),
                      dict(table_width=(1 << 24) - 1, table_stride=1 << 24, page_size=128), dict(num_pages=1, heads_kv=65537), dict(tokens=0x7ffffffe)]


def calls(lib, c):
    a = _lib.Fa8KvAttentionParams(cache=c, q=FAKE, q_token_stride=256, q_head_stride=64, o=FAKE, dtype=0, heads=4, is_causal=1, softmax_scale=0.125)
    return (lib.fa8_kv_append(ctypes.byref(c), FAKE, 128, 64, FAKE, 128, 64, 0, None),
            lib.fa8_kv_read(ctypes.byref(c), FAKE, FAKE, 0, None), lib.fa8_kv_attention(ctypes.byref(a), None))


def test_every_declared_symbol_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO_DIR, "include", "fa8_kv_cache.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(fa8_[a-z_0-9]+)\s*\(", text))
    assert declared == set(_lib.KV_SYMBOLS)
    raw = ctypes.CDLL(LIB_PATH)
    for name in declared:
        assert hasattr(raw, name), name
    assert _lib.load().fa8_kv_version() == 100
    assert b"page number" in _lib.load().fa8_error_string(_lib.FA8_ERR_BAD_INDEX)


@pytest.mark.parametrize("kw", BAD_CACHES, ids=str)
def test_bad_cache_descriptions_are_refused(kw):
    assert set(calls(_lib.load(), cache_params(**kw))) == {_lib.FA8_ERR_BAD_ARG}


@pytest.mark.parametrize("kw", UNSUPPORTED_CACHES, ids=str)
def test_unsupported_caches_are_refused(kw):
    assert set(calls(_lib.load(), cache_params(**kw))) == {_lib.FA8_ERR_UNSUPPORTED}


def test_bad_rows_are_refused():
    lib, c = _lib.load(), cache_params()
    bad = _lib.FA8_ERR_BAD_ARG
    assert lib.fa8_kv_append(None, FAKE, 128, 64, FAKE, 128, 64, 0, None) == bad
    for rows in ((None, 128, 64, FAKE, 128, 64), (FAKE, 128, 64, None, 128, 64), (FAKE + 2, 128, 64, FAKE, 128, 64), (FAKE, 129, 64, FAKE, 128, 64),
                 (FAKE, 128, 64, FAKE, 128, 60), (FAKE, -128, 64, FAKE, 128, 64), (FAKE, 128, 64, FAKE, 128, -64)):
        assert lib.fa8_kv_append(ctypes.byref(c), *rows, 0, None) == bad
    assert lib.fa8_kv_append(ctypes.byref(c), FAKE, 128, 64, FAKE, 128, 64, 2, None) == bad
    for out in ((None, FAKE, 0), (FAKE, None, 0), (FAKE + 8, FAKE, 0), (FAKE, FAKE, 3)):
        assert lib.fa8_kv_read(ctypes.byref(c), *out, None) == bad
    good = dict(cache=c, q=FAKE, q_token_stride=256, q_head_stride=64, o=FAKE, dtype=0, heads=4, is_causal=1, softmax_scale=0.125)
    assert lib.fa8_kv_attention(None, None) == bad
    for kw in (dict(q=None), dict(o=None), dict(q=FAKE + 8), dict(o=FAKE + 8), dict(q_token_stride=4), dict(q_head_stride=-64), dict(dtype=5),
               dict(heads=0), dict(heads=3), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(lse=FAKE + 2)):
        assert lib.fa8_kv_attention(ctypes.byref(_lib.Fa8KvAttentionParams(**{**good, **kw})), None) == bad, kw
    for args in ((0, 1, 1, 1, 64, 16, 1, 148), (1, -1, 1, 1, 64, 16, 1, 148), (1, 1, 3, 2, 64, 16, 1, 148), (1, 1, 1, 1, 64, 16, 1, 0)):
        assert lib.fa8_kv_attention_workspace(*args) == bad


def test_rows_past_32_bits_are_unsupported():
    c = cache_params(tokens=1 << 24, batch=2)
    p = _lib.Fa8KvAttentionParams(cache=c, q=FAKE, q_token_stride=64 * 128, q_head_stride=64, o=FAKE, dtype=0, heads=128, is_causal=1, softmax_scale=0.125)
    assert _lib.load().fa8_kv_attention(ctypes.byref(p), None) == _lib.FA8_ERR_UNSUPPORTED


@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 3), (7, 100), (64, 64), (1000, 1000), (2, 5000)])
@pytest.mark.parametrize("heads,heads_kv,head_dim", [(1, 1, 32), (32, 8, 128), (160, 1, 64), (9, 3, 256)])
def test_workspace_is_a_matter_of_sizes(batch, tokens, heads, heads_kv, head_dim):
    """Never negative, and bounded: a partial result for each of the GPU's warps, or sixteen of the output."""
    lib = _lib.load()
    for width in (1, 40, 5000):
        n = lib.fa8_kv_attention_workspace(batch, tokens, heads, heads_kv, head_dim, 64, width, 148)
        assert 0 <= n <= max(148 * 18 * 32 * (head_dim + 2) * 4 + 8192, 16 * tokens * heads * (head_dim + 2) * 4)
        assert n == lib.fa8_kv_attention_workspace(batch, tokens, heads, heads_kv, head_dim, 64, width, 148)


def test_no_tokens_is_no_launch():
    assert set(calls(_lib.load(), cache_params(tokens=0))) == {_lib.FA8_OK}


def test_host_tensors_are_refused():
    c = PagedKVCache(torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn), torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn), torch.ones(2, 1), torch.ones(2, 1))
    x, t, s = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv_append(c, x, x, t, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv_read(c, t, s, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        flash_attention_paged_kv(x, c, t, s)


def test_oracle_scales():
    assert po.scale_for(448.0, 448.0) == 1.0 and po.scale_for(448.5, 448.0) == 2.0 and po.scale_for(3.5, 448.0) == 2.0 ** -7
    assert po.scale_for(0.0, 448.0) == 2.0 ** -64 and po.scale_for(1e30, 448.0) == 2.0 ** 64


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_oracle_append_in_pieces_keeps_what_one_piece_keeps(dtype):
    """Rounding anew by a power of two changes only what becomes subnormal: here nothing, so token by token and all at
    once give the same values."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 1, 32, generator=g).half()
    x = torch.where(x.abs() < 0.1, torch.full_like(x, 0.5), x)
    x[7] *= 16
    cache = [torch.zeros(2, 1, 16, 32).to(dtype), torch.zeros(2, 1, 16, 32).to(dtype), torch.zeros(2, 1), torch.zeros(2, 1)]
    table = torch.tensor([[1, 0]])
    whole = po.append(cache, x, x, table, [20])
    for i in range(20):
        cache = po.append(cache, x[i:i + 1], x[i:i + 1], table, [i + 1])
    for a, b in zip(po.keys_values(whole, table, 0, 20), po.keys_values(cache, table, 0, 20)):
        assert torch.equal(a, b)
    assert torch.equal(whole[2], cache[2])


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(4)
    cache = [torch.randn(3, 2, 16, 32, generator=g).to(torch.float8_e4m3fn), torch.randn(3, 2, 16, 32, generator=g).to(torch.float8_e4m3fn),
             torch.tensor([[1.0, 2.0], [0.5, 1.0], [4.0, 0.25]]), torch.ones(3, 2)]
    table = torch.tensor([[2, 0, -1], [1, -1, -1]])
    q = torch.randn(5, 4, 32, generator=g).half()
    o, lse, _ = po.attention(q, cache, table, [20, 1], True, 0.3, [0, 3, 5])
    k, v = po.keys_values(cache, table, 0, 20)
    for i in range(3):
        for h in range(4):
            s = (k[:18 + i, h // 2] @ q[i, h].double()) * 0.3
            torch.testing.assert_close(o[i, h], torch.softmax(s, 0) @ v[:18 + i, h // 2])
            torch.testing.assert_close(lse[i, h], torch.logsumexp(s, 0))
    assert bool((o[3] == 0).all()) and bool((lse[3] == -float("inf")).all())              # one key, two new tokens: the first sees none
    torch.testing.assert_close(o[4, 0], po.keys_values(cache, table, 1, 1)[1][0, 0])


def test_every_status_is_declared_for_callers_of_the_forward_alone(tmp_path):
    """fa8_fwd and fa8_check_status return what a call of the paged cache left in the status words they share, so its code is in their
    header, with the value that the package uses; the other header adds to it."""
    import shutil
    import subprocess
    names = {n: v for n, v in vars(_lib).items() if n == "FA8_OK" or n.startswith("FA8_ERR_")}
    assert names["FA8_ERR_BAD_INDEX"] == -5
    text = open(os.path.join(REPO_DIR, "include", "fa8_b200.h")).read()
    for name, value in names.items():
        assert re.search(rf"#define {name} \(?{value}\)?\s", text), name
    about = re.findall(r"/\*(.*?)\*/\s*(?:int|const char\*|int64_t) (fa8_\w+)\(", text, flags=re.S)
    for function in ("fa8_fwd", "fa8_check_status"):
        assert any("FA8_ERR_BAD_INDEX" in words for words, name in about if name == function), function
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    for headers in (["fa8_b200.h"], ["fa8_kv_cache.h"], ["fa8_kv_cache.h", "fa8_b200.h"]):
        source = "".join(f'#include "{h}"\n' for h in headers) + "int code = FA8_ERR_BAD_INDEX;\n"
        (tmp_path / "c.c").write_text(source)
        subprocess.run([cc, "-Wall", "-Werror", "-std=c99", "-I" + os.path.join(REPO_DIR, "include"), "-c", str(tmp_path / "c.c"),
                        "-o", str(tmp_path / "c.o")], check=True)
