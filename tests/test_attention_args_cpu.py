"""The attention operators without a device: the argument checks that run before anything reaches the GPU
(csrc/attention_args.h, compiled into a host program with address and undefined-behaviour checks), the shapes the
Python binding refuses, and the Rust bindings and calls against the header."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

import strata_cuda as sc
import test_crate_ffi_cpu as ffi
from test_crate_sequence_cpu import body, code, pieces

ROOT = Path(__file__).resolve().parents[1]
NAMES = {"strata_kv_cache", "strata_kv_append", "strata_attention"}


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_argument_checks(tmp_path):
    exe = tmp_path / "attention_args_check"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           "-I", str(ROOT / "strata-rs_b200" / "csrc"), str(ROOT / "tests" / "attention_args_check.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def cache(**change):
    return sc.KvCache(**{**dict(k_ptr=1 << 20, v_ptr=1 << 30, table_ptr=1 << 16, len_ptr=1 << 17, n_pages=10, page_size=16, n_kv_head=2, head_dim=64, max_pages=8), **change})


def shape(**change):
    return sc.Attention(**{**dict(n_seq=2, n_head=4, scale=0.1, seq_len=3), **change})


def test_offsets_must_match_the_sequences():
    for make in (lambda o: sc.Attention(3, 4, 0.1, offsets=o), lambda o: sc.KvAppend(3, 4, 64, offsets=o)):
        make([0, 1, 2, 3])
        with pytest.raises(sc.BackendError) as e:
            make([0, 1, 2])
        assert e.value.code == sc.ERR_INVALID


@pytest.mark.parametrize("bad", [dict(n_seq=0), dict(n_head=3), dict(n_head=0), dict(seq_len=-1), dict(q_stride=5), dict(o_stride=-8), dict(offsets=[0, 5, 4]),
                                 dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=1e-60), dict(scale=1e60),
                                 dict(dtype=sc.F16)])
def test_work_bytes_refuses_bad_shapes(bad):
    assert sc.attention_work_bytes(shape(), cache()) > 0
    with pytest.raises(sc.BackendError) as e:
        sc.attention_work_bytes(shape(**bad), cache())
    assert e.value.code == (sc.ERR_UNSUPPORTED_QUANT if "dtype" in bad else sc.ERR_INVALID)


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(head_dim=12), dict(head_dim=264), dict(page_size=0), dict(page_size=24), dict(n_pages=0), dict(max_pages=0),
                                 dict(max_pages=1 << 28), dict(table_stride=7), dict(token_stride=64), dict(token_stride=132), dict(head_stride=56),
                                 dict(page_stride=1000), dict(n_kv_head=0), dict(n_kv_head=3)])
def test_work_bytes_refuses_bad_caches(bad):
    with pytest.raises(sc.BackendError) as e:
        sc.attention_work_bytes(shape(), cache(**bad))
    assert e.value.code == sc.ERR_INVALID


def test_the_workspace_does_not_grow_with_the_lengths():
    one = sc.attention_work_bytes(shape(), cache())
    assert one == sc.attention_work_bytes(shape(n_seq=1000, seq_len=1), cache(n_pages=1 << 20, max_pages=1 << 20)) < 32 << 20
    assert sc.attention_work_bytes(shape(seq_len=0), cache()) == 0


def test_rust_bindings_match_the_header(monkeypatch):
    """ffi_attention.rs declares strata_attention.h's functions and structs, as ffi.rs does the other headers'."""
    monkeypatch.setattr(ffi, "HEADERS", [ROOT / "include" / "strata_attention.h"])
    monkeypatch.setattr(ffi, "FFI", ffi.CRATE / "src" / "ffi_attention.rs")
    monkeypatch.setattr(ffi, "C_TO_RUST", {**ffi.C_TO_RUST, **{n: n for n in NAMES}})
    c, r = ffi.c_functions(), ffi.rust_functions()
    assert len(c) == 4 and c == r
    cs, rs = ffi.c_structs(), ffi.rust_structs()
    assert set(cs) == NAMES and cs == rs
    text = code("attention.rs")
    for name, (_, params) in r.items():
        calls = [m.end() - 1 for m in re.finditer(name + r"\(", text)]
        assert len(calls) == 1 and len(pieces(body(text, calls[0]))) == len(params), name
    for name, fields in rs.items():
        made = [m.end() - 1 for m in re.finditer(r"(?<!-> )\b" + name + r" \{", text)]
        assert len(made) == 1, name
        assert [p.split(":")[0].strip() for p in pieces(body(text, made[0]))] == [f[0] for f in fields], name
    assert {"mod ffi_attention;", "pub mod attention;"} <= set(code("lib.rs").split("\n"))
    for fn in ("kv_append", "attention", "logprobs"):
        assert f"pub unsafe fn {fn}(" in text
    for brackets in ("()", "{}", "[]"):
        assert text.count(brackets[0]) == text.count(brackets[1])


def test_python_structs_match_the_header(monkeypatch):
    monkeypatch.setattr(ffi, "HEADERS", [ROOT / "include" / "strata_attention.h"])
    monkeypatch.setattr(ffi, "C_TO_RUST", {**ffi.C_TO_RUST, **{n: n for n in NAMES}})
    cs = ffi.c_structs()
    for name, made in (("strata_kv_cache", sc.KvCacheDesc), ("strata_kv_append", sc.KvAppendDesc), ("strata_attention", sc.AttentionDesc)):
        assert [f[0] for f in cs[name]] == [f[0] for f in made._fields_]
