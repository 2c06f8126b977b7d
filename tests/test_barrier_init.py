"""Kernels' barriers in shared memory, by reading their sources: a thread that initialises them is no warp's whole, so the block meets once, whatever branches it takes, before
anything waits for them or has the tensor cores signal them (the thread that initialised them may signal them and load before)."""

import pathlib
import re

import pytest

SOURCES = sorted(p for p in (pathlib.Path(__file__).resolve().parents[1] / "rl_b200" / "csrc").glob("*.cu") if "mbar_init(" in p.read_text())
USES = re.compile(r"\b(mbar_wait|mbar_try_wait|one_wait|warp_wait|wait_long|umma_commit\w*)\s*\(")
MEETS = re.compile(r"__syncthreads\(\);|\bcluster_sync\(\);")


def _kernels(text):
    """(name, body) of each kernel, without comments."""
    text = re.sub(r"//[^\n]*|__(?:launch_bounds|cluster_dims)__\([^\n]*?\)(?=\s*(?:\w|\n))", "", text)
    for m in re.finditer(r"__global__\s[^;{]*?(\w+)\s*\([^{;]*\)\s*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end() : at - 1]


def _met_before_use(body):
    """Whether behind the last initialisation a statement of the body's own level, which no branch leaves out, joins the block before the first use."""
    at = max(m.end() for m in re.finditer(r"mbar_init\(", body))
    use = USES.search(body, at)
    end = use.start() if use else len(body)
    for m in MEETS.finditer(body, at, end):
        before = body[: m.start()]
        alone = re.search(r"[;}]\s*$", before)      # (not what an `if` without brackets guards)
        if before.count("{") == before.count("}") and alone:
            return True
    return False


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_blocks_meet_between_barriers_first_state_and_their_use(path):
    found = [(name, body) for name, body in _kernels(path.read_text()) if "mbar_init(" in body]
    assert found
    for name, body in found:
        assert _met_before_use(body), f"{path.name}: {name} uses barriers that some path has not seen initialised"


def test_reading_sees_a_branch_that_does_not_meet():
    first = "if (t == 0) { mbar_init(a, 1); } "
    assert _met_before_use(first + "pdl_sync(); __syncthreads(); mbar_wait(a, 0);")
    for rest in ("mbar_wait(a, 0); __syncthreads();", "if (x) { __syncthreads(); } mbar_wait(a, 0);", "if (x) __syncthreads(); mbar_wait(a, 0);",
                 "if (warp != 0) { bar_sync(1, 160); } umma_commit(a);"):
        assert not _met_before_use(first + rest)
