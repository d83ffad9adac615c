"""Kernels that may start while the one before them still runs (they call after_previous) read what that one wrote: their sources have none of the
loads that take memory for constant over a kernel's whole life."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mimir_b200", "csrc")


def block(text, at, opening="{", closing="}"):
    """From the next opening bracket behind `at` to the one that closes it."""
    start = text.index(opening, at)
    depth, i = 0, start
    while True:
        depth += (text[i] == opening) - (text[i] == closing)
        i += 1
        if not depth:
            return text[start:i], i


def without_comments(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def functions(text):
    """(name, whether it is a kernel, parameters, body) of the functions that run on the device."""
    for m in re.finditer(r"__(global|device)__", text):
        head = next(h for h in re.compile(r"\b(\w+)\s*(?=\()").finditer(text, m.end()) if not h[1].startswith("__"))
        params, end = block(text, head.end(), "(", ")")
        behind = text[end:].lstrip()
        if behind.startswith("{"):
            yield head[1], m[1] == "global", params, block(text, end)[0]


def test_no_loads_of_read_only_memory():
    found = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        text = without_comments(open(path).read())
        if "after_previous()" not in text or os.path.basename(path) == "common.cuh":
            continue
        all_of = list(functions(text))
        bodies = {}
        for name, _, _, body in all_of:
            bodies[name] = bodies.get(name, "") + body
        for name, kernel, params, body in all_of:
            if not kernel or "after_previous()" not in body:
                continue
            found += 1
            assert not re.search(r"const\s+[\w:]+\s*\*\s*__restrict__", params), (path, name)
            seen, left = set(), [name]
            while left:                                      # the kernel, and what it calls
                f = left.pop()
                if f not in seen:
                    seen.add(f)
                    left += [c for c in re.findall(r"\b(\w+)\s*(?:<[\w\s,]*>)?\s*\(", bodies[f]) if c in bodies]
            for f in seen:
                assert "__ldg(" not in bodies[f] and "ld.global.nc" not in bodies[f], (path, name, f)
    assert found >= 9        # the products, two sums of parts, join, scoring, probabilities, three of the clipping
