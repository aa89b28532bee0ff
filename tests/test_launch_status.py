"""CPU: no entry point reports success before it has asked whether its launches failed.

Read from the sources: a launch that fails leaves its error behind, and whoever asks next would take it for one of
their own.  In every function that launches and returns a status, KH_LAUNCHED() lies between a launch and `return KH_OK`."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).parent.parent / "klearu_amd" / "csrc"
SOURCES = sorted(p.name for p in CSRC.glob("*.hip"))


def functions(text):
    """(name, whether it returns a status, body) of the file's functions."""
    text = re.sub(r"//[^\n]*", "", text)
    head = re.compile(r"^(?:extern \"C\" |static |inline )*(int|void)\s+(\w+)\([^;{]*\)\s*\{", re.M)
    for m in head.finditer(text):
        end = text.index("\n}", m.end())
        yield m[2], m[1] == "int", text[m.end():end]


def unreported(text):
    """Names of functions that return KH_OK with a launch's error unasked for."""
    found = list(functions(text))
    quiet = [name for name, status, body in found if not status and "hipLaunchKernelGGL" in body]
    while True:  # void functions that call those
        more = [n for n, status, body in found if not status and n not in quiet and
                any(re.search(rf"\b{q}\b\s*(<[^;()]*>)?\(", body) for q in quiet)]
        if not more:
            break
        quiet += more
    step = re.compile(r"(?P<launch>hipLaunchKernelGGL" + "".join(rf"|\b{q}\b" for q in quiet) +
                      r")|(?P<asks>KH_LAUNCHED\(\)|hipGetLastError\(\))|(?P<ok>return KH_OK)")
    for name, status, body in found:
        open_ = False
        for m in step.finditer(body) if status else ():
            if m["ok"] and open_:
                yield name
                break
            open_ = open_ if m["ok"] else bool(m["launch"])


def test_the_rule_itself():
    ok = "static int f(int n) {\n  hipLaunchKernelGGL(k, g);\n  KH_LAUNCHED();\n  return KH_OK;\n}\n"
    early = "static int f(int n) {\n  hipLaunchKernelGGL(k, g);\n  if (n) return KH_OK;\n  KH_LAUNCHED();\n  return KH_OK;\n}\n"
    other = "static void h(int n) {\n  hipLaunchKernelGGL(k, g);\n}\nint f(int n) {\n  h(n);\n  return KH_OK;\n}\n"
    assert [list(unreported(t)) for t in (ok, early, other)] == [[], ["f"], ["f"]]


@pytest.mark.parametrize("source", SOURCES)
def test_launches_are_asked_for(source):
    assert list(unreported((CSRC / source).read_text())) == []
