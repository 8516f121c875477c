"""The 4-bit GEMM's stage hand-over in compiled code, on the CPU.

A step's plane fragments are direct-to-LDS loads issued three steps before other
waves read them; the wave that issued them waits, before the step's barrier, until
at most n of its loads are in flight, n being what it issued after them: the loads
of the two steps before. Loads of a value that nothing reads are not in the
compiled code, and a count that included them would let the fragments still be in
flight. Checked on every path through every form of the kernel."""

from __future__ import annotations

import re
import subprocess

import pytest

import helpers

HIPCC = "/opt/rocm/bin/hipcc"


def hand_overs(body):
    """(fewest loads issued in the two steps before on any path, vmcnt allowed) of each
    barrier that a wait leads up to. What comes before the first barrier is one step."""
    at = {m.group(1): i for i, m in enumerate(re.match(r"(\.LBB\w+):", s) for s in body) if m}
    # the fewest counts suffice: a path with no fewer loads in both steps shows nothing new
    best, found, todo = {}, {}, [(0, 0, 0, None)]
    while todo:
        i, before, issued, allowed = todo.pop()
        while i < len(body):
            if re.match(r"\.LBB", body[i]):
                known = best.setdefault((i, allowed), [])
                if any(p <= before and q <= issued for p, q in known):
                    break
                known.append((before, issued))
            s = body[i]
            op = s.split()[0] if s.split() else ""
            if re.match(r"(global|buffer)_load_", op):
                issued, allowed = issued + 1, None
            elif op == "s_waitcnt" and "vmcnt" in s:
                allowed = int(re.search(r"vmcnt\((\d+)\)", s).group(1))
            elif op == "s_barrier":
                if allowed is not None:
                    two = before + issued
                    found[i] = min(found.get(i, (two, allowed)), (two, allowed))
                before, issued, allowed = issued, 0, None
            elif op.startswith("s_cbranch"):
                todo.append((at[s.split()[1]], before, issued, allowed))
            elif op == "s_branch":
                i = at[s.split()[1]]
                continue
            elif op == "s_endpgm":
                break
            i += 1
    return [found[i] for i in sorted(found)]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "mx4_linear.s"
    csrc = helpers.PKG_DIR / "csrc"
    subprocess.run(
        [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature",
         "-Xclang", "-packed-fp32-ops", f"-I{helpers.REPO / 'include'}", f"-I{csrc}", "-x", "hip",
         "--cuda-device-only", "-S", str(csrc / "kernels" / "mx4_linear.hip"), "-o", str(out)],
        check=True, capture_output=True, timeout=300)
    return {m.group(1): [s.strip() for s in m.group(2).splitlines()]
            for m in re.finditer(r"^(_Z\S*mx4_gemm_kernel\S*):(.*?)^\.Lfunc_end", out.read_text(),
                                 re.M | re.S)}


def test_every_hand_over_waits_for_the_planes_it_hands_over(kernels):
    assert len(kernels) >= 4, sorted(kernels)
    for name, body in kernels.items():
        steps = hand_overs(body)
        assert len(steps) >= 8, name  # two chunks of four steps in the loop at least
        for i, (issued, allowed) in enumerate(steps):
            assert allowed <= issued, f"{name}, step {i}: {issued} loads issued, {allowed} allowed in flight"


def test_the_check_sees_a_dropped_load():
    """The check itself, on a listing: a step that allows more than was issued."""
    ok = ["buffer_load_x lds"] * 9 + ["s_waitcnt vmcnt(6)", "s_barrier"] + [
        "buffer_load_x lds", "s_waitcnt vmcnt(1)", "s_barrier", "buffer_load_x lds",
        "s_waitcnt vmcnt(2)", "s_barrier", "s_endpgm"]
    assert all(a <= n for n, a in hand_overs(ok))
    bad = ok[:-3] + ["s_waitcnt vmcnt(3)", "s_barrier", "s_endpgm"]
    assert not all(a <= n for n, a in hand_overs(bad))
