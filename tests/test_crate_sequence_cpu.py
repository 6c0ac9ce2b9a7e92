"""The crate's public calls of the sequence operators (crates/strata-backend-cuda/src/sequence.rs): every binding of
ffi_sequence.rs is called there, with as many arguments, every field of its structs is set, and the types' numbers are
the header's. Parsed as text, as there is no Rust toolchain here."""
import re

import test_crate_ffi_cpu as ffi

SRC = ffi.CRATE / "src"
INCLUDE = ffi.ROOT / "include"


def code(name):
    return re.sub(r"//[^\n]*", "", (SRC / name).read_text())


def body(text, at):
    """What the bracket at `at` encloses."""
    depth = 0
    for i in range(at, len(text)):
        depth += text[i] in "({["
        depth -= text[i] in ")}]"
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError("unbalanced brackets")


def pieces(text):
    """The top-level comma-separated pieces of `text`."""
    out, depth = [""], 0
    for ch in text:
        depth += ch in "({["
        depth -= ch in ")}]"
        if ch == "," and depth == 0:
            out.append("")
        else:
            out[-1] += ch
    return [p.strip() for p in out if p.strip()]


def test_every_binding_is_called(monkeypatch):
    monkeypatch.setattr(ffi, "FFI", SRC / "ffi_sequence.rs")
    bound, text = ffi.rust_functions(), code("sequence.rs")
    assert len(bound) == 4
    for name, (_, params) in bound.items():
        calls = [m.end() - 1 for m in re.finditer(name + r"\(", text)]
        assert len(calls) == 1, name
        assert len(pieces(body(text, calls[0]))) == len(params), name
    for name, fields in ffi.rust_structs().items():
        made = [m.end() - 1 for m in re.finditer(r"(?<!-> )\b" + name + r" \{", text)]
        assert len(made) == 1, name
        assert [p.split(":")[0].strip() for p in pieces(body(text, made[0]))] == [f[0] for f in fields], name


def test_they_can_be_reached():
    lib, text = code("lib.rs"), code("sequence.rs")
    assert "pub mod sequence;" in lib
    assert "dead_code" not in code("ffi_sequence.rs")
    for fn in ("short_conv", "gated_delta", "sample"):
        assert f"pub unsafe fn {fn}(" in text
    assert "pub fn work_bytes(" in text and "pub fn synchronize(" in text
    for brackets in ("()", "{}", "[]"):
        assert text.count(brackets[0]) == text.count(brackets[1])


def test_the_types_numbers_are_the_headers():
    c = ffi.c_constants()
    text = code("sequence.rs")
    assert f"Self::F32 => {c['STRATA_QUANT_F32']}" in text and f"Self::Bf16 => {c['STRATA_QUANT_BF16']}" in text
