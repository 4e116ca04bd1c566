"""Refusals of the 8-bit KV cache and token scoring operators, on the CPU:
every bad argument is an error before any device work, empty calls do nothing.
The addresses are numbers that no call here may follow."""
import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest

from orator_b200 import _lib, ops
from oracle import kv_quant_oracle as O

A = 4096  # an aligned address


def cache(**kw):
    a = dict(pool=A, pages=8, Hkv=8, Dh=128, fmt=ops.KVQ_INT8, page_table=A, seqs=2, max_pages=4)
    a.update(kw)
    return ops.KvQuantCache(**a)


BAD_CACHES = [dict(pool=0), dict(pool=A + 4), dict(pages=0), dict(pages=(1 << 27) + 1), dict(Hkv=0),
              dict(Hkv=1025), dict(Dh=96), dict(Dh=0), dict(fmt=2), dict(fmt=-1), dict(page_table=0),
              dict(seqs=-1), dict(seqs=65537), dict(max_pages=0), dict(max_pages=1 << 27), dict(seqs=65536, max_pages=1 << 15), dict(seqs=65536, max_pages=(1 << 15) - 1)]


def write(c, **kw):
    a = dict(k=A, v=A, dtype=0, k_stride=1024, v_stride=1024, row_seq=A, row_pos=A, rows=3)
    a.update(kw)
    ops.KvQuantWrite(c, **a)


def read(c, **kw):
    a = dict(k=A, v=A, dtype=0, k_stride=1024, v_stride=1024, row_seq=A, row_pos=A, rows=3)
    a.update(kw)
    ops.KvQuantRead(c, **a)


def attend(c, **kw):
    a = dict(q=A, out=A, dtype=1, q_stride=2048, out_stride=2048, lse=0, lens=A, Hq=16, q_tokens=1,
             shared=0, shared_pages=0, scale=0.1, workspace=A, workspace_bytes=1 << 40)
    a.update(kw)
    ops.KvQuantAttention(c, **a)


def score(**kw):
    a = dict(logits=A, dtype=0, rows=2, vocab=100, row_stride=100, targets=A, top=3, logprob=A,
             entropy=A, top_ids=A, top_logprobs=A)
    a.update(kw)
    ops.TokenLogprobs(**a)


def refused(f, *a, **kw):
    with pytest.raises(_lib.OrxError) as e:
        f(*a, **kw)
    assert e.value.code == 1 and len(str(e.value)) > len("orx error 1: "), e.value


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
@pytest.mark.parametrize("call", [write, read, attend])
def test_bad_cache(call, bad):
    refused(call, cache(**bad))


@pytest.mark.parametrize("bad", [dict(k=0), dict(v=0), dict(dtype=2), dict(dtype=-1), dict(k_stride=1023),
                                 dict(v_stride=0), dict(row_seq=0), dict(row_pos=0),
                                 dict(rows=(1 << 25) + 1)], ids=str)
@pytest.mark.parametrize("call", [write, read])
def test_bad_rows(call, bad):
    refused(call, cache(), **bad)


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(dtype=3), dict(q_stride=2047), dict(out_stride=-1),
                                 dict(lens=0), dict(Hq=0), dict(Hq=12), dict(q_tokens=0), dict(q_tokens=4097),
                                 dict(shared_pages=1), dict(shared=A, shared_pages=5), dict(shared=A, shared_pages=-1),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace=0),
                                 dict(workspace=A + 8), dict(workspace_bytes=0)], ids=str)
def test_bad_attention(bad):
    refused(attend, cache(), **bad)


@pytest.mark.parametrize("name", ["k", "v", "row_seq", "row_pos", "q", "out", "lens", "lse", "shared", "logits", "targets", "logprob", "entropy",
                                  "top_ids", "top_logprobs", "page_table", "err"])
def test_addresses_between_elements(name):
    """An address that is no multiple of its elements' size is refused before anything else looks at it."""
    for off, dtype in ((1, 1), (2, 0), (1, 0)):
        kw, c = {name: A + off}, cache()
        if name in ("page_table", "err"):
            c, kw = cache(**kw), {}
        if name in ("k", "v", "row_seq", "row_pos", "page_table", "err"):
            refused(write, c, dtype=dtype, **kw)
            refused(read, c, dtype=dtype, **kw)
        if name in ("q", "out", "lens", "lse", "shared", "page_table", "err"):
            refused(attend, c, dtype=dtype, **dict(dict(shared=A, shared_pages=1), **kw))
        if name in ("logits", "targets", "logprob", "entropy", "top_ids", "top_logprobs"):
            refused(score, dtype=dtype, **kw)


def test_too_many_query_rows():
    refused(attend, cache(seqs=65536), Hq=16, q_tokens=4096, q_stride=2048)
    refused(ops.KvQuantAttentionWorkspace, cache(seqs=65536), 16, 4096)


def test_too_much_work():
    """Work whose shares could not be counted: 2^41 (page, kv head, 8 query rows) or more, in its own pages or in shared ones."""
    most = (1 << 27) - 1
    for c, kw in ((dict(seqs=1, max_pages=most), dict(Hq=512, q_tokens=4096, q_stride=1 << 16, out_stride=1 << 16)),
                  (dict(seqs=1, max_pages=most, Hkv=1), dict(Hq=1024, q_tokens=256, q_stride=1 << 17, out_stride=1 << 17)),
                  (dict(seqs=4096, max_pages=500000), dict(Hq=64, q_tokens=1024, q_stride=1 << 13, out_stride=1 << 13, shared=A, shared_pages=400000))):
        refused(attend, cache(**c), **kw)
        args = kw["Hq"], kw["q_tokens"], kw.get("shared_pages", 0)
        refused(ops.KvQuantAttentionWorkspace, cache(**c), *args)
    for c, args in ((dict(seqs=1, max_pages=most, Hkv=1), (8, 4, 0)), (dict(seqs=1, max_pages=most, Hkv=1), (512, 8, 1000)),
                    (dict(seqs=65536, max_pages=32000), (8, 1, 0)), (dict(seqs=4096, max_pages=500000), (16, 4, 10))):
        assert ops.KvQuantAttentionWorkspace(cache(**c), *args) > 0


@pytest.mark.parametrize("bad", [dict(logits=0), dict(dtype=2), dict(vocab=0), dict(vocab=-5), dict(vocab=(1 << 19) + 1, row_stride=1 << 20), dict(rows=(1 << 24) + 1), dict(row_stride=99),
                                 dict(top=-1), dict(top=33), dict(vocab=2, top=3), dict(targets=0), dict(top_ids=0),
                                 dict(top_logprobs=0)], ids=str)
def test_bad_scores(bad):
    refused(score, **bad)


def test_empty_calls_do_nothing():
    for c in (cache(), cache(seqs=0)):
        write(c, rows=0, k=0)
        read(c, rows=-1, v=0)
    attend(cache(seqs=0), q=0, out=0, lens=0)
    score(rows=0, logits=0)


def test_null_cache():
    for name, n in (("orx_kvq_write", 8), ("orx_kvq_read", 8)):
        with pytest.raises(_lib.OrxError):
            _lib.call(name, None, A, A, 0, 1024, 1024, A, A, 1, None)
    with pytest.raises(_lib.OrxError):
        _lib.call("orx_kvq_attention_workspace", C.byref(cache()), 16, 1, 0, None)


def test_sizes():
    assert [ops.KvQuantBlockBytes(d) for d in (64, 128, 96, 0, -64)] == [2176, 4224, 0, 0, 0]
    assert all(O.block_bytes(d) == ops.KvQuantBlockBytes(d) for d in (64, 128))
    n = [ops.KvQuantAttentionWorkspace(cache(seqs=s), 16, t, p) for s, t, p in ((0, 1, 0), (1, 1, 0), (64, 1, 4), (64, 8, 4))]
    assert n == sorted(n) and n[0] > 0


def test_oracle_quantiser():
    """Values on codes come back exactly; any other value within half a step of its row's scale."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    for fmt, half in ((O.INT8, 0.5), (O.E4M3, 16.0)):
        c, s = O.quantise(x, fmt)
        # the quotient is rounded once more (2^-24 of at most 448)
        assert (np.abs(c * s[:, None].astype(np.float64) - x) <= (half + 448 * 2.0**-24) * s[:, None]).all()
        again, s2 = O.quantise((c * s[:, None]).astype(np.float32), fmt)
        assert (again == c).all()
    for bad in (np.nan, np.inf, -np.inf):
        c, s = O.quantise(np.array([[1, bad]], np.float32), O.INT8)
        assert np.isnan(s).all() and (c == 0).all()
    c, s = O.quantise(np.array([[1e-40, 0]], np.float32), O.E4M3)
    assert s[0] == 0 and (c == 0).all()


CPP = r"""
#include <cstdio>
#include "orator_b200/asr_ops.h"
using namespace orator::model;
int main() {
  orx_kvq c = {};
  c.pool = (void*)4096; c.page_table = (const int*)4096;
  c.pages = 8; c.kv_heads = 8; c.head_dim = 128; c.seqs = 2; c.max_pages = 4;
  int thrown = 0;
  try { asr_ops::KvQuantWrite(c, nullptr, nullptr, 0, 1024, 1024, nullptr, nullptr, 1); } catch (const std::runtime_error&) { ++thrown; }
  try { asr_ops::KvQuantRead(c, nullptr, nullptr, 0, 1024, 1024, nullptr, nullptr, 1); } catch (const std::runtime_error&) { ++thrown; }
  try { asr_ops::KvQuantAttention(c, nullptr, nullptr, 0, 2048, 2048, nullptr, nullptr, 16, 1, nullptr, 0, 1.f, nullptr, 0); } catch (const std::runtime_error&) { ++thrown; }
  try { asr_ops::TokenLogprobs(nullptr, 0, 1, 10, 10, nullptr, 0, nullptr, nullptr, nullptr, nullptr); } catch (const std::runtime_error&) { ++thrown; }
  asr_ops::KvQuantWrite(c, nullptr, nullptr, 0, 1024, 1024, nullptr, nullptr, 0);
  std::printf("%d %d\n", thrown, asr_ops::KvQuantAttentionWorkspace(c, 16, 1) > 0);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_cpp_header(tmp_path):
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    if not os.path.exists(os.path.join(cuda, "include", "cuda_runtime_api.h")):
        pytest.skip("CUDA headers not found")
    src, exe, lib = tmp_path / "a.cc", tmp_path / "a", os.path.dirname(_lib.LIB_PATH)
    src.write_text(CPP)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(root, "include"), "-I",
                    os.path.join(cuda, "include"), str(src), "-o", str(exe), "-L", lib, "-l:liborator_b200.so",
                    f"-Wl,-rpath,{lib}"], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout.split() == ["4", "1"]
