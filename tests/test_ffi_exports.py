"""rust/llm-ffi/src/sampler.rs exports what a C caller needs of each operator
around the sampling call, without a Rust compiler: an `llm_*` function for each
method of the binding, with the method's arguments behind the handle, passed on
in order."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FFI = os.path.join(ROOT, "rust", "llm-ffi", "src", "sampler.rs")
BINDING = os.path.join(ROOT, "rust", "llm-kernel", "src", "hip_sampler.rs")


def source(path):  # (read by the tests: the module is also imported where the file is not)
    with open(path) as f:
        return f.read()


def parameters(path, name):
    """(name, type) of each parameter of a function, its result and its body."""
    m = re.search(r'\n( *)pub (?:unsafe )?(?:extern "C" )?fn %s\(([^)]*)\)\s*->\s*([^{]+?)\s*\{\n(.*?)\n\1\}\n'
                  % name, source(path), flags=re.S)
    assert m, name
    params = [tuple(x.strip() for x in p.split(":")) for p in m.group(2).split(",") if ":" in p]
    return params, m.group(3), m.group(4)


@pytest.mark.parametrize("method", ["process_logits", "logprobs", "pages_update", "pages_compact", "pages_copy"])
def test_each_method_is_exported(method):
    want, _, _ = parameters(BINDING, method)
    got, result, body = parameters(FFI, "llm_" + method)
    assert result == "i32" and got[0] == ("sampler", "*mut c_void")
    # references are pointers on the C side
    assert got[1:] == [(n, re.sub(r"^&", "*const ", t)) for n, t in want]
    passed = re.search(r"\.%s\(([^)]*)\)" % method, body).group(1)
    names = [a.strip().lstrip("&*") for a in passed.split(",")]
    assert names == [n for n, _ in want]
    # what is behind a reference is checked before it is read
    for name in ["sampler"] + [n for n, t in want if t.startswith("&")]:
        assert f"{name}.is_null()" in body
    assert re.search(r'#\[no_mangle\]\npub unsafe extern "C" fn llm_%s\(' % method, source(FFI))


def test_the_size_of_a_cache_s_work_array_is_exported():
    """0 stands for sizes that are refused."""
    want, _, _ = parameters(BINDING, "pages_work_words")
    got, result, body = parameters(FFI, "llm_pages_work_words")
    assert got == want and result == "u64"
    assert "pages_work_words(rows, num_pages).unwrap_or(0)" in body
    assert re.search(r'#\[no_mangle\]\npub extern "C" fn llm_pages_work_words\(', source(FFI))
    used = re.search(r"use llm_kernel::hip_sampler::\{(.*?)\};", source(FFI), flags=re.S).group(1)
    assert "pages_work_words" in [x.strip() for x in used.split(",")]
