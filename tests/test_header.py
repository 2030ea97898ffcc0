"""The public header's conventions: whole comments, and what they promise (no GPU)."""
import re
from pathlib import Path

HEADER = (Path(__file__).resolve().parent.parent / "include" / "baracuda_kernels.h").read_text()


def test_comment_lines_are_whole():
    for comment in re.findall(r"/\*.*?\*/", HEADER, re.S):
        for line in comment.split("\n")[1:]:
            assert re.match(r" \*(/| |$)", line), line


def test_conventions_say_what_a_workspace_is_for():
    text = " ".join(HEADER[:HEADER.index("#ifndef")].replace(" *", " ").split())
    assert "split along K (two launches, bit-identical output)" in text
    assert "Without it every entry point but those two runs as-is" in text
