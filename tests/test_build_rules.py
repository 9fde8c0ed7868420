"""Rules that the compiler does not check: what inline assembly says that it changes."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "spla_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.rglob("*") if p.suffix in (".hip", ".hpp", ".cpp"))


def _assembly(text):
    """(template, rest) of every asm statement: the string literals up to the first colon outside of them, the operands behind it"""
    for m in re.finditer(r"\basm\s+volatile\s*\(|\basm\s*\(", text):
        at, depth, parts, template = m.end(), 1, [], None
        while depth:
            if text[at] == '"':
                end = re.compile(r'"(?:\\.|[^"\\])*"').match(text, at).end()
                parts.append(text[at:end])
                at = end
                continue
            if text[at] == ":" and template is None:
                template, parts = "".join(parts), []
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            parts.append(text[at])
            at += 1
        yield (template, "".join(parts)) if template is not None else ("".join(parts), "")


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_assembly_that_writes_m0_says_so(path):
    """the compiler keeps values of its own in M0 and merges equal ones: it has to know every other writer"""
    for template, rest in _assembly(path.read_text()):
        if re.search(r"\bs_\w+\s+m0\s*,", template):
            assert '"m0"' in rest, template


def test_the_rule_finds_the_statements():
    text = 'asm volatile("s_mov_b32 m0, %0" ::"s"(f(x)) : "memory");  asm("" : "+v"(y));  asm volatile("s_nop 3")'
    assert list(_assembly(text)) == [('"s_mov_b32 m0, %0" ', '::"s"(f(x)) : "memory")'), ('"" ', ': "+v"(y))'), ('"s_nop 3")', "")]


SWITCH = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _strings(text):
    return re.findall(r'"((?:\\.|[^"\\])*)"', text)


def test_both_compilers_build_without_packed_fp32_arithmetic():
    """the library's kernels (build.py) and the ones around user-defined ops, which are compiled at run time (jit.hip)"""
    ahead = _strings(re.search(r"cmd \+= \[f\"--offload-arch=.*?\]", (CSRC.parent / "build.py").read_text()).group())
    at_run_time = _strings(re.search(r"opts\[\]\s*=\s*\{.*?\};", (CSRC / "kernels" / "jit.hip").read_text(), re.S).group())
    assert ahead[-4:] == SWITCH
    assert at_run_time[-4:] == SWITCH
