"""The operators around the sampling call (llmk_process_logits, llmk_logprobs,
llmk_pages_*) without a GPU: the ctypes and Rust structs have the C layout, and
every call that cannot be right is refused before a device is touched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import llmk
from llmk import _lib
from llmk import sampler as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HDR = os.path.join(ROOT, "include", "llmk_sampler.h")
RS = os.path.join(ROOT, "rust", "llm-kernel", "src", "hip_sampler.rs")

STRUCTS = [("llmk_process_logits_args", _lib.ProcessLogitsArgs, "LlmkProcessLogitsArgs"),
           ("llmk_logprobs_args", _lib.LogprobsArgs, "LlmkLogprobsArgs"),
           ("llmk_page_cache", _lib.PageCacheArgs, "LlmkPageCache")]


@pytest.mark.parametrize("name,mirror,_rust", STRUCTS)
def test_ctypes_structs_match_the_c_layout(tmp_path, name, mirror, _rust):
    fields = [f for f, _ in mirror._fields_]
    body = "".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields)
    (tmp_path / "l.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "llmk_sampler.h"\n'
                                  "int main(void){\n" + body +
                                  f'  printf("SIZE %zu\\n", sizeof({name}));\n  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"),
                    str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for f in fields:
        assert int(got[f]) == getattr(mirror, f).offset, f
    assert int(got["SIZE"]) == ctypes.sizeof(mirror)


C2RS = {"const void*": "*const c_void", "void*": "*mut c_void", "int32_t": "i32", "uint32_t": "u32",
        "uint64_t": "u64", "float": "f32", "const float*": "*const f32", "float*": "*mut f32",
        "const int32_t*": "*const i32", "const uint32_t*": "*const u32", "uint32_t*": "*mut u32",
        "const uint64_t*": "*const u64"}


@pytest.mark.parametrize("name,mirror,rust", STRUCTS)
def test_rust_structs_match_the_header(name, mirror, rust):
    src = re.sub(r"/\*.*?\*/", "", open(HDR).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, src, flags=re.S).group(1)
    c = []
    for d in body.split(";"):
        d = " ".join(d.split())
        if d:
            m = re.match(r"(.*?)\s*\b([a-z_]+)$", d)
            c.append((m.group(2), C2RS[m.group(1).replace(" *", "*").strip()]))
    rbody = re.search(r"pub struct %s \{(.*?)\n\}" % rust, open(RS).read(), flags=re.S).group(1)
    assert c == [(n, t.strip()) for n, t in re.findall(r"pub ([a-z_]+): ([^,]+),", rbody)]
    assert [n for n, _ in c] == [f for f, _ in mirror._fields_]


# A handle that no check may look into: all of them come before the device.
FAKE = ctypes.create_string_buffer(4096)
H = ctypes.cast(FAKE, ctypes.c_void_p)
P = 0x10000


def _process(**kw):
    a = _lib.ProcessLogitsArgs()
    base = dict(logits=P, dtype=_lib.LLMK_F32, batch=2, vocab=100, row_stride=100, out=P * 16,
                out_dtype=_lib.LLMK_F32, out_stride=100)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return _lib.load().llmk_process_logits(H, ctypes.byref(a), None)


BAD = _lib.LLMK_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw,code,word", [
    (dict(vocab=0), _lib.LLMK_ERR_EMPTY_LOGITS, "Empty"),
    (dict(logits=None), BAD, "required"),
    (dict(out=None), BAD, "required"),
    (dict(dtype=3), BAD, "dtype"),
    (dict(out_dtype=7), BAD, "dtype"),
    (dict(out_dtype=_lib.LLMK_BF16), BAD, "out_dtype"),
    (dict(dtype=_lib.LLMK_F16, out_dtype=_lib.LLMK_BF16), BAD, "out_dtype"),
    (dict(row_stride=99), BAD, "stride"),
    (dict(out_stride=99), BAD, "stride"),
    (dict(logits=P + 2), _lib.LLMK_ERR_ALIGNMENT, "aligned"),
    (dict(out=P * 16 + 1), _lib.LLMK_ERR_ALIGNMENT, "aligned"),
    (dict(softcap=-1.0), BAD, "softcap"),
    (dict(softcap=float("nan")), BAD, "softcap"),
    (dict(softcap=float("inf")), BAD, "softcap"),
    (dict(hist_offsets=P), BAD, "go together"),
    (dict(hist_lengths=P), BAD, "need hist_offsets"),
    (dict(hist_counts=P), BAD, "need hist_offsets"),
    (dict(extra_begin=P, extra_count=P), BAD, "go together"),
    (dict(extra_tokens=P), BAD, "go together"),
    (dict(bias_offsets=P, bias_values=P), BAD, "go together"),
    (dict(allow_mask=P, mask_words_per_row=3, mask_rows=2), BAD, "mask_words_per_row"),
    (dict(allow_mask=P, mask_words_per_row=4, mask_rows=1), BAD, "mask_index"),
    (dict(mask_index=P), BAD, "needs allow_mask"),
    (dict(row_seq=P), BAD, "sequences"),
    (dict(vocab=2**31, row_stride=2**31, out_stride=2**31), _lib.LLMK_ERR_CAPACITY, "vocab"),
    # rows written over rows that are read
    (dict(out=P + 4), BAD, "overlaps"),
    (dict(out=P, out_stride=101), BAD, "overlaps"),
    (dict(out=P, dtype=_lib.LLMK_BF16), BAD, "overlaps"),
    (dict(out=P + 400, row_stride=150, out_stride=150), BAD, "overlaps"),
    (dict(batch=2**31 - 1, vocab=2**20, row_stride=2**20, out_stride=2**20, out=P),
     _lib.LLMK_ERR_CAPACITY, "too large"),
])
def test_process_logits_refuses(kw, code, word):
    assert _process(**kw) == code
    assert word in _lib.last_error()


def test_calls_with_nothing_to_do():
    lib = _lib.load()
    assert _process(batch=0) == 0
    a = _lib.LogprobsArgs()
    a.logits, a.vocab, a.row_stride, a.tokens, a.out_logprobs = P, 8, 8, P, P
    assert lib.llmk_logprobs(H, ctypes.byref(a), None) == 0
    assert lib.llmk_pages_copy(H, 1, P, 64, 8, 0, None, None, None) == 0
    assert lib.llmk_pages_copy(H, 0, None, 0, 8, 4, P, P, None) == 0


def test_null_handles_and_args():
    lib = _lib.load()
    for call in (lambda s: lib.llmk_process_logits(s, None, None),
                 lambda s: lib.llmk_logprobs(s, None, None),
                 lambda s: lib.llmk_pages_update(s, None, P, P, P, None),
                 lambda s: lib.llmk_pages_compact(s, None, P, None)):
        for s in (None, H):
            assert call(s) == BAD
            assert "NULL" in _lib.last_error()
    assert lib.llmk_pages_copy(None, 1, P, 64, 8, 1, P, P, None) == BAD
    assert lib.llmk_pages_work_words(1, 1, None) == BAD


@pytest.mark.parametrize("kw,code,word", [
    (dict(vocab=0), _lib.LLMK_ERR_EMPTY_LOGITS, "Empty"),
    (dict(logits=None), BAD, "required"),
    (dict(dtype=9), BAD, "dtype"),
    (dict(row_stride=7), BAD, "stride"),
    (dict(logits=P + 1), _lib.LLMK_ERR_ALIGNMENT, "aligned"),
    (dict(softcap=-2.0), BAD, "softcap"),
    (dict(tokens=None), BAD, "nothing"),
    (dict(out_logprobs=None), BAD, "out_logprobs"),
    (dict(top_n=33), _lib.LLMK_ERR_CAPACITY, "top_n"),
    (dict(top_n=5, out_top_ids=P), BAD, "out_top"),
    (dict(vocab=2**20 + 1, row_stride=2**21), _lib.LLMK_ERR_CAPACITY, "vocab"),
])
def test_logprobs_refuses(kw, code, word):
    a = _lib.LogprobsArgs()
    base = dict(logits=P, dtype=_lib.LLMK_F32, batch=2, vocab=8, row_stride=8, tokens=P, out_logprobs=P)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    assert _lib.load().llmk_logprobs(H, ctypes.byref(a), None) == code
    assert word in _lib.last_error()


@pytest.mark.parametrize("kw,code,word", [
    (dict(rows=0), BAD, "rows"),
    (dict(num_pages=0), BAD, "num_pages"),
    (dict(rows=2**20 + 1), _lib.LLMK_ERR_CAPACITY, "rows"),
    (dict(num_pages=2**25 + 1), _lib.LLMK_ERR_CAPACITY, "num_pages"),
    (dict(max_pages=0), BAD, "max_pages"),
    (dict(page_tokens=0), BAD, "page_tokens"),
    (dict(max_pages=2**20, page_tokens=2**11), _lib.LLMK_ERR_CAPACITY, "2^31"),
    (dict(table=None), BAD, "required"),
    (dict(used=None), BAD, "required"),
    (dict(work=P + 4), _lib.LLMK_ERR_ALIGNMENT, "work"),
    (dict(n_pools=65536), _lib.LLMK_ERR_CAPACITY, "n_pools"),
    (dict(n_pools=1, page_bytes=0), BAD, "page_bytes"),
    (dict(n_pools=1, page_bytes=64, pools=None), BAD, "pools"),
    (dict(n_pools=1, page_bytes=2**40 + 1), _lib.LLMK_ERR_CAPACITY, "page_bytes"),
])
def test_pages_refuse(kw, code, word):
    lib = _lib.load()
    a = _lib.PageCacheArgs()
    base = dict(rows=4, max_pages=8, page_tokens=16, num_pages=64, table=P, lengths=P, refs=P, used=P,
                work=P, n_pools=0, page_bytes=0, pools=P)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    for rc in (lib.llmk_pages_update(H, ctypes.byref(a), P, P, P, None),
               lib.llmk_pages_compact(H, ctypes.byref(a), P, None)):
        assert rc == code
        assert word in _lib.last_error()


def test_pages_calls_need_their_outputs():
    lib = _lib.load()
    a = _lib.PageCacheArgs()
    for k, v in dict(rows=4, max_pages=8, page_tokens=16, num_pages=64, table=P, lengths=P, refs=P,
                     used=P, work=P).items():
        setattr(a, k, v)
    assert lib.llmk_pages_update(H, ctypes.byref(a), None, None, P, None) == BAD
    assert "nothing" in _lib.last_error()
    assert lib.llmk_pages_update(H, ctypes.byref(a), P, P, None, None) == BAD
    assert lib.llmk_pages_compact(H, ctypes.byref(a), None, None) == BAD
    assert lib.llmk_pages_copy(H, 1, P, 64, 8, 1, None, P, None) == BAD
    assert lib.llmk_pages_copy(H, 1, None, 64, 8, 1, P, P, None) == BAD


def test_work_words_grow_with_the_cache():
    lib = _lib.load()
    w = ctypes.c_uint64()
    seen = []
    for rows, pages in ((1, 1), (64, 1000), (1 << 20, 1000), (64, 1 << 25)):
        assert lib.llmk_pages_work_words(rows, pages, ctypes.byref(w)) == 0
        assert w.value >= 4 * pages + rows  # the lists of pages, an entry per row
        seen.append(w.value)
    assert seen == sorted(seen)


# ---- the Python wrappers' own checks, on host tensors ------------------------

def test_python_wrappers_refuse_host_tensors_and_wrong_types():
    lb = llmk.LogitsBatch(logits=torch.zeros(2, 8))
    with pytest.raises(S.SamplerError, match="CUDA"):
        S._process_args(lb, torch.zeros(2, 8))
    with pytest.raises(S.SamplerError, match="float32, bfloat16 or float16"):
        S._process_args(llmk.LogitsBatch(logits=torch.zeros(2, 8, dtype=torch.float64)), torch.zeros(2, 8))
    with pytest.raises(S.SamplerError, match="unit stride"):
        S._process_args(llmk.LogitsBatch(logits=torch.zeros(8, 2).t()), torch.zeros(2, 8))
    with pytest.raises(S.SamplerError, match="vocab 9"):
        S._process_args(llmk.LogitsBatch(logits=torch.zeros(2, 8), vocab=9), torch.zeros(2, 9))
    with pytest.raises(S.SamplerError, match="out must be"):
        S._process_args(lb, torch.zeros(3, 8))
    with pytest.raises(S.SamplerError, match="CUDA"):
        llmk.PagePools([torch.zeros(4, 8)])
    with pytest.raises(S.SamplerError, match="no pools"):
        llmk.PagePools([])
