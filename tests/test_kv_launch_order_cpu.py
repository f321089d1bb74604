"""Kernels that are launched beside the one before them wait for it on every way out.

What follows such a kernel in its stream is ordered behind that kernel alone: where all its blocks could return
without the wait, the next call could read what the kernel before has not written yet."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "go-fann_b200" / "csrc"


def kernels(text):
    """{name: body} of the __global__ functions of a source file."""
    found = {}
    for m in re.finditer(r"__global__[^{;]*?(\w+)\s*\((?:[^()]|\([^()]*\))*\)\s*\{", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text)):
        src = m.string
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(src[at], 0)
            at += 1
        found[m.group(1)] = src[m.end() : at]
    return found


def dependents():
    got = []
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        if "ProgrammaticStreamSerialization" not in text:
            continue
        body = kernels(text)
        launched = set()
        for call in re.findall(r"cudaLaunchKernelEx\(&cfg,\s*(\w+)", text):
            if call in body:
                launched.add(call)
            else:  # a variable that names the variants
                launched |= {n for n in re.findall(r"\w+", re.search(rf"auto {call} =(.*?);", text, re.S).group(1)) if n in body}
        got += [pytest.param(body[n], id=f"{path.stem}-{n}") for n in sorted(launched)]
    return got


def test_there_are_dependent_kernels():
    assert len(dependents()) >= 4


@pytest.mark.parametrize("body", dependents())
def test_every_return_is_behind_the_wait(body):
    # lambdas return values of their own: only a kernel's return has none
    # one at the outer level covers all that follows it, one elsewhere only the return right behind it
    outer = next((m.start() for m in re.finditer(r"wait_previous\(\);", body)
                  if body[: m.start()].count("{") == body[: m.start()].count("}")), None)
    assert outer is not None, "no wait that every thread reaches"
    for m in re.finditer(r"\breturn\s*;", body[:outer]):
        assert re.search(r"wait_previous\(\);\s*$", body[: m.start()]), body[max(0, m.start() - 200) : m.end()]


@pytest.mark.parametrize("body", dependents())
def test_results_of_the_kernel_before_come_from_l2(body):
    """Its blocks may still run beside this kernel, so a plain load could be served by the read-only path or by a line
    that they left in L1."""
    sources = {"scores", "parts"}
    while True:  # names of pointers into the scratch
        names = "|".join(sources)
        more = set(re.findall(rf"const float\* (\w+) = (?:{names})\b", body)) - sources
        if not more:
            break
        sources |= more
    for name in sources:
        assert not re.search(rf"\b{name}\s*\[", body), f"{name} is indexed"
        assert not re.search(rf"(?<!float)\*\s*(?:reinterpret_cast<[^>]*>)?\(?{name}\b", body), f"{name} is read through"
