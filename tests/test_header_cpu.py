"""The public header as its readers have it: whole comments, and the contract of the operators on MX blocks."""
import os
import re
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include", "ptwm_mi355x.h")


@pytest.fixture(scope="module")
def text():
    with open(HEADER) as f:
        return f.read()


def test_comments_are_whole(text):
    """A comment of several lines has a star before each, or stands in a column behind a declaration."""
    for comment in re.findall(r"/\*.*?\*/", text, re.S):
        for line in comment.split("\n")[1:]:
            assert re.match(r" \*( |$|/)|  ", line), line


def test_contract_of_the_operators(text):
    """What holds for all operators of the section stands before the first of them."""
    start = text.index("3. Operators on microscaled (MX) blocks")
    said = re.sub(r"\s*\n \*\s*", " ", text[start:text.index("ptwm_mi355x_rms_norm_mx_cuda(")])
    for words in ("return without waiting for it", "hold no state, lock or workspace of their own", "allocate nothing",
                  "may be captured into a graph", "alignment of their elements only", "strides are between rows",
                  "Returns 0; -1 for arguments that do not fit together"):
        assert words in said, words


def test_header_is_c(text, tmp_path):
    c = tmp_path / "h.c"
    c.write_text(f'#include "{os.path.abspath(HEADER)}"\nint main(void) {{ return 0; }}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-Wcomment", "-fsyntax-only", str(c)], check=True)
