"""The 4-bit GEMM's stage hand-over in compiled code, on the CPU.

A step's plane fragments (three loads a wave) are direct-to-LDS loads that other
waves read after the next barrier; the wave that issued them waits, before that
barrier, until at most n of its loads are in flight. Loads complete in order, so what
may still be in flight is the newest n: among them may be the planes of the two steps
after the one handed over, six direct loads, and of three steps (nine) at the first
barrier, which hands over the first of four steps. Loads of a value that nothing reads
are not in the compiled code, and a count that included them would let a seventh be in
flight. Checked on every path through every form of the kernel."""

from __future__ import annotations

import re
import subprocess

import pytest

import helpers

HIPCC = "/opt/rocm/bin/hipcc"


WINDOW = 32  # newest loads remembered: more than any wait allows


def hand_overs(body):
    """For each barrier that a wait for loads leads up to, in program order: the most
    direct loads among the newest n issued, n being what the wait allows, over all paths."""
    at = {m.group(1): i for i, m in enumerate(re.match(r"(\.LBB\w+):", s) for s in body) if m}
    found, seen, todo = {}, set(), [(0, "", None)]
    while todo:
        i, recent, allowed = todo.pop()
        while i < len(body):
            s = body[i]
            if s.startswith(".LBB"):
                if (i, recent, allowed) in seen:
                    break
                seen.add((i, recent, allowed))
            op = s.split()[0] if s.split() else ""
            if re.match(r"(global|buffer)_load_", op):
                recent = (recent + ("d" if s.endswith(" lds") else "r"))[-WINDOW:]
                allowed = None
            elif op == "s_waitcnt" and "vmcnt" in s:
                allowed = int(re.search(r"vmcnt\((\d+)\)", s).group(1))
                assert allowed < WINDOW
            elif op == "s_barrier":
                if allowed is not None:
                    direct = recent[len(recent) - min(allowed, len(recent)):].count("d")
                    found[i] = max(found.get(i, 0), direct)
                allowed = None
            elif op.startswith("s_cbranch"):
                todo.append((at[s.split()[1]], recent, allowed))
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
    assert len(kernels) >= 6, sorted(kernels)  # three widths, with and without RMSNorm
    for name, body in kernels.items():
        steps = hand_overs(body)
        assert len(steps) >= 13, name  # the first, two chunks in the loop, one at the end
        assert steps[0] <= 9, f"{name}: first hand-over leaves {steps[0]} direct loads in flight"
        for i, direct in enumerate(steps[1:]):
            assert direct <= 6, f"{name}, step {i}: {direct} direct loads may be in flight"


def test_the_check_sees_a_dropped_load():
    """The check itself, on listings: the weights' two loads between the planes', then
    the same without them and with the same count."""
    planes = ["buffer_load_dwordx4 v0, s[0:3], 0 offen lds"] * 3
    weights = ["buffer_load_dwordx4 v[0:3], v4, s[0:3], 0 offen"] * 2
    end = ["s_waitcnt vmcnt(8)", "s_barrier", "s_endpgm"]
    assert hand_overs(planes + planes + weights + planes + end) == [6]
    assert hand_overs(planes + planes + planes + end) == [8]
