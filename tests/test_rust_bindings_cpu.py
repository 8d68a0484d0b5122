"""The Rust crate's declarations against the header they are of (no Rust compiler here: read as text): every function declared with
as many parameters, and every operator's entry point called by a wrapper of the crate."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "integration", "crates", "hodu_rocm_kernels", "src")


def parameters(text):
    """{function: number of parameters} of `name(.., ..)` declarations"""
    out = {}
    for name, args in re.findall(r"\b(hodu_rocm_\w+)\s*\(([^()]*)\)", text):
        args = args.strip().rstrip(",")
        out.setdefault(name, 0 if args in ("", "void") else args.count(",") + 1)
    return out


def source(name):
    text = open(os.path.join(SRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def header():
    return parameters(subprocess.check_output(["gcc", "-E", "-P", f"-I{ROOT}/include", os.path.join(ROOT, "include", "hodu_rocm_kernels.h")], text=True))


def test_declarations_have_the_headers_parameters():
    want = header()
    got = {name: n for name, n in parameters("\n".join(re.findall(r"pub fn [^;]*;", source("ffi.rs")))).items()}
    assert len(got) > 25
    for name, n in got.items():
        assert name in want and want[name] == n, (name, n, want.get(name))


def test_every_operator_has_a_wrapper():
    called = set(re.findall(r"ffi::(hodu_rocm_\w+)", source("kernels.rs") + source("context.rs")))
    for name in ("softmax", "softmax_masked", "attention", "attention_masked", "sum", "cast", "contiguous", "paged_plan", "paged_store", "attention_varlen",
                 "attention_paged", "ctx_stream", "ctx_set_stream"):
        assert f"hodu_rocm_{name}" in called, name


def test_wrappers_pass_as_many_arguments_as_are_declared():
    want, text = header(), source("kernels.rs")
    for m in re.finditer(r"ffi::(hodu_rocm_\w+)\s*\(", text):
        depth, args, i = 1, 1, m.end()
        while depth:
            ch = text[i]
            depth += (ch in "([{") - (ch in ")]}")
            args += ch == "," and depth == 1
            i += 1
        assert want[m.group(1)] == args, (m.group(1), args, want[m.group(1)])
