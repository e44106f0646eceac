"""The operators' host checks at the ends of their arguments' ranges, without a
GPU.  Each call runs in a process of its own: what a check lets through must not
end the caller's."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CALL = """
import ctypes, sys
sys.path.insert(0, {pkg!r})
from llmk import _lib
lib = _lib.load()
handle = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)
a = _lib.{struct}()
for k, v in {fields!r}.items():
    setattr(a, k, v)
rc = lib.{function}(handle, ctypes.byref(a), None)
print(rc, _lib.last_error())
"""

P = 0x10000
PROCESS = dict(logits=P, dtype=0, batch=2, vocab=100, row_stride=100, out=P * 16, out_dtype=0, out_stride=100)
LOGPROBS = dict(logits=P, dtype=0, batch=2, vocab=8, row_stride=8, tokens=P, out_logprobs=P)


def call(function, struct, fields):
    code = CALL.format(pkg=os.path.join(ROOT, "llm-rs_amd"), struct=struct, function=function, fields=fields)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    rc, _, message = r.stdout.strip().partition(" ")
    return int(rc), message


def process(**kw):
    return call("llmk_process_logits", "ProcessLogitsArgs", dict(PROCESS, **kw))


def logprobs(**kw):
    return call("llmk_logprobs", "LogprobsArgs", dict(LOGPROBS, **kw))


@pytest.mark.parametrize("kw", [dict(row_stride=2**62, out=P + 4, out_stride=2**62),
                                dict(row_stride=2**63, out=P + 4, out_stride=2**63),
                                dict(row_stride=2**54 + 1), dict(out_stride=2**54 + 1)])
def test_strides_whose_bytes_overflow_are_refused(kw):
    rc, message = process(**kw)
    assert rc == -3 and "2^55" in message
    if "out_stride" not in kw:
        rc, message = logprobs(**kw)
        assert rc == -3 and "2^55" in message


# 256 threads a row, or 512 where a row has 40 tiles of 1024 logits and a top list
@pytest.mark.parametrize("kw", [dict(batch=2**32 - 1), dict(batch=2**32 - 512), dict(batch=2**24),
                                dict(batch=2**23, vocab=40960, row_stride=40960, top_n=1, out_top_ids=P,
                                     out_top_logprobs=P)])
def test_logprobs_of_more_rows_than_a_grid_holds(kw):
    rc, message = logprobs(**kw)
    assert rc == -3 and "too large" in message


@pytest.mark.parametrize("kw", [dict(batch=2**24, vocab=8, row_stride=8, out_stride=8, out=2**40),
                                dict(batch=2**22, vocab=4 * 4096, row_stride=2**15, out_stride=2**15, out=2**50),
                                dict(batch=2**32 - 1, vocab=1, row_stride=1, out_stride=1, out=2**40)])
def test_process_logits_of_more_segments_than_a_grid_holds(kw):
    rc, message = process(**kw)
    assert rc == -3 and "too large" in message


@pytest.mark.parametrize("cap", [1e-45, 2.0**-129, 1.1754942e-38])
def test_softcaps_whose_reciprocal_may_overflow_are_refused(cap):
    for f in (process, logprobs):
        rc, message = f(softcap=cap)
        assert rc == -1 and "softcap" in message
