"""Rows of floats in LDS that the attention kernels over caches in 4 bits store and load four at a time: a row's pitch has to keep every one of
them on 16 bytes, which the type promises the compiler.  Read off the sources, no kernel runs here."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "flh_amd" / "csrc"
SOURCES = ["decode_attention_i4.hip", "prefill_attention_i4.hip"]


def constants(text, d):
    """The integer constants of struct Layout that depend on D alone."""
    body = text[text.index("struct Layout {"):]
    found = {"D": d}
    for name, value in re.findall(r"\b(k\w+) = ([^,;]+)", body[:body.index("};")]):
        if re.fullmatch(r"[D\d\s+*/]+", value):
            found[name] = eval(value.replace("/", "//"), {"D": d})     # (digits, D and signs alone)
    return found


def pitches(text):
    """Names of the pitches by which a row is multiplied in an access to four floats."""
    for access in re.findall(r"\(\s*(?:const\s+)?v4f\s*\*\s*\)\s*\(([^;]*)\)", text):
        yield from re.findall(r"\w+\s*\*\s*(?:L::)?(k[A-Z]\w*|D)\b", access)


@pytest.mark.parametrize("source", SOURCES)
@pytest.mark.parametrize("d", [64, 128])
def test_pitches_are_multiples_of_sixteen_bytes(source, d):
    text = (CSRC / source).read_text()
    known, used = constants(text, d), set(pitches(text))
    assert used
    for name in used:
        assert known[name] % 4 == 0, (source, name, known[name])


def test_the_reader_sees_them():
    text = "struct Layout {\n  static constexpr int kA = D + 2, kB = D * 2 + 4;\n};\n*(v4f*)(x + col * L::kA + 16 * i) = y; v = *(const v4f*)(f + r * L::kB);"
    assert set(pitches(text)) == {"kA", "kB"} and constants(text, 64) == {"D": 64, "kA": 66, "kB": 132}
