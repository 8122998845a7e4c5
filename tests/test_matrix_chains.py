"""What the compiler makes of chains of matrix instructions, from its assembly (no GPU).

An instruction of 16 places that takes up, in the same registers, the sums that the one of 32
places right before it leaves misses that product in its first two rows of four.  The compiler
puts no wait between the two (it does where such sums are another operand), so no kernel may
chain instructions of different shapes without one."""

from __future__ import annotations

import importlib.util
import re
import subprocess
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "gdn-state-codec_amd"
WAITS = 8  # states: what the compiler keeps before sums are read as another operand
PRODUCT = re.compile(r"(v_mfma\w+) ([av]\[\d+:\d+\]), (\S+), (\S+), ([av]\[\d+:\d+\]|\S+)")


def reads(operands: str, sums: str) -> bool:
    """Whether an operand has a register of `sums`."""
    def registers(text):
        return {(kind, i) for kind, first, last in re.findall(r"([av])\[?(\d+):?(\d*)", text)
                for i in range(int(first), int(last or first) + 1)}

    return bool(registers(operands) & registers(sums))


def close_chains(assembly: str) -> list[str]:
    """Pairs of different instructions, the second adding to the first's sums, with less than
    WAITS wait states between them."""
    found, last = [], []  # (instruction, its sums, wait states since)
    for line in assembly.splitlines():
        line = line.strip()
        if re.match(r"[\w$.]+:", line):  # a label: what came before is another path's, too
            continue
        if not line or line[0] in ".;":
            continue
        product = PRODUCT.match(line)
        if product:
            name, to, left, right, taken = product.groups()
            for other, sums, waits in reversed(last):
                if sums == taken:
                    if other != name and waits < WAITS and not reads(left + right, sums):
                        found.append(f"{other} -> {name} after {waits}: {line}")
                    break
        nop = re.match(r"s_nop (\d+)", line)
        waits = int(nop[1]) + 1 if nop else 0 if line.startswith("s_waitcnt") else 1
        last = [(n, s, w + waits) for n, s, w in last if w + waits < WAITS]
        if product:
            last.append((name, to, 0))
    return found


def test_the_pattern_is_found():
    close = """
	v_mfma_f32_16x16x32_bf16 v[6:9], v[50:53], v[10:13], v[6:9]
	s_waitcnt lgkmcnt(1)
	v_mfma_f32_16x16x16_bf16 v[6:9], v[36:37], v[30:31], v[6:9]
"""
    assert len(close_chains(close)) == 1
    assert not close_chains(close.replace("s_waitcnt lgkmcnt(1)", "s_nop 7"))
    assert not close_chains(close.replace("16x16x16", "16x16x32"))
    assert not close_chains(close.replace("v[30:31], v[6:9]", "v[30:31], 0"))


@pytest.mark.parametrize("source", ["draft_tree.hip", "delta_prepare.hip"])
def test_chains_of_different_shapes_wait(source, tmp_path):
    """The sources that use more than one shape."""
    spec = importlib.util.spec_from_file_location("package_build", PACKAGE / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    out = tmp_path / "kernel.s"
    subprocess.run([build.HIPCC, *build.COMMON_FLAGS, "--offload-device-only", "-S",
                    str(build.CSRC / source), "-o", str(out)], check=True, capture_output=True)
    assembly = out.read_text()
    assert len(set(re.findall(r"v_mfma\w+", assembly))) > 1
    assert close_chains(assembly) == []
