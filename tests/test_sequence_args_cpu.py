"""The sequence operators without a device: the argument checks that run before
anything reaches the GPU (csrc/sequence_args.h, compiled into a host program
with address and undefined-behaviour checks), the shapes the Python binding
refuses, and the Rust bindings against the header."""
import shutil
import subprocess
from pathlib import Path

import pytest

import strata_cuda as sc
import test_crate_ffi_cpu as ffi

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_argument_checks(tmp_path):
    exe = tmp_path / "sequence_args_check"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           "-I", str(ROOT / "strata-rs_b200" / "csrc"), str(ROOT / "tests" / "sequence_args_check.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_offsets_must_match_the_sequences():
    for make in (lambda o: sc.ShortConv(3, 8, 4, offsets=o), lambda o: sc.GatedDelta(3, 1, 1, 8, 8, offsets=o)):
        make([0, 1, 2, 3])
        with pytest.raises(sc.BackendError) as e:
            make([0, 1, 2])
        assert e.value.code == sc.ERR_INVALID


@pytest.mark.parametrize("bad", [dict(n_seq=0), dict(n_k_head=3), dict(k_dim=257), dict(v_dim=0), dict(seq_len=-1),
                                 dict(q_stride=5), dict(offsets=[0, 5, 4]), dict(offsets=[-1, 5, 6]), dict(dtype=sc.F16),
                                 dict(scale=float("nan")), dict(l2_eps=float("nan"))])
def test_work_bytes_refuses_bad_shapes(bad):
    shape = dict(n_seq=2, n_k_head=2, n_v_head=4, k_dim=64, v_dim=64, seq_len=7)
    sc.gated_delta_work_bytes(sc.GatedDelta(**shape))
    with pytest.raises(sc.BackendError) as e:
        sc.gated_delta_work_bytes(sc.GatedDelta(**{**shape, **bad}))
    assert e.value.code == (sc.ERR_UNSUPPORTED_QUANT if "dtype" in bad else sc.ERR_INVALID)


def test_one_token_needs_no_workspace():
    for n in (1, 64, 1000):
        assert sc.gated_delta_work_bytes(sc.GatedDelta(n, 16, 32, 128, 128, seq_len=1)) == 0


def test_rust_bindings_match_the_header(monkeypatch):
    """ffi_sequence.rs declares strata_sequence.h's functions and structs, as ffi.rs does the other headers'."""
    monkeypatch.setattr(ffi, "HEADERS", [ROOT / "include" / "strata_sequence.h"])
    monkeypatch.setattr(ffi, "FFI", ffi.CRATE / "src" / "ffi_sequence.rs")
    monkeypatch.setattr(ffi, "C_TO_RUST", {**ffi.C_TO_RUST, "strata_short_conv": "strata_short_conv",
                                           "strata_gated_delta": "strata_gated_delta"})
    c, r = ffi.c_functions(), ffi.rust_functions()
    assert len(c) == 4 and set(c) == set(r)
    assert {n: (ret, args) for n, (ret, args) in c.items()} == r
    cs, rs = ffi.c_structs(), ffi.rust_structs()
    assert set(cs) == set(rs) == {"strata_short_conv", "strata_gated_delta"}
    assert cs == rs
    assert "mod ffi_sequence;" in (ffi.CRATE / "src" / "lib.rs").read_text()
