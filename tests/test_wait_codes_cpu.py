"""The codes that a kernel reports when a barrier wait ran out: one range for each kernel's file, so that a code names it."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "uzu_b200" / "csrc"


def _ranges():
    found = {}
    for path in sorted(CSRC.glob("*.cu")):
        if path.name == "decode_mega.cu":      # (words of its own)
            continue
        for line in path.read_text().splitlines():
            if "gave_up" in line or "report_wait_error" in line or "watch" in line:
                for code in re.findall(r"\b0x([1-9a-f])[0-9a-f]{2}u\b", line):
                    found.setdefault(code, set()).add(path.name)
    return found


def test_a_code_names_its_kernel():
    found = _ranges()
    assert len(found) >= 5 and all(len(files) == 1 for files in found.values()), found


def test_the_list_says_so():
    text = (CSRC / "wait_errors.h").read_text()
    for code, files in _ranges().items():
        assert f"0x{code}xx {next(iter(files))}" in text, (code, files)
