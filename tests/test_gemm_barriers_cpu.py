"""The product's pipeline barriers, walked on the CPU: whichever role gives up,
and wherever, the barrier that holds tensor memory back has completed no phase
before its own commit."""

import ctypes
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
FULL, EMPTY, ACC_FULL, ACC_EMPTY, DRAINED, BYTES = range(6)
FORMS = [(8, 2), (6, 2), (6, 1)]


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    out = tmp_path_factory.mktemp("probe") / "gemm_barriers.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-o", str(out),
                    str(ROOT / "tests" / "gemm_barriers_probe.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    return lib.probe_barrier


def kinds(stages, acc):
    return ([(FULL, s) for s in range(stages)] + [(EMPTY, s) for s in range(stages)]
            + [(ACC_FULL, a) for a in range(acc)] + [(ACC_EMPTY, a) for a in range(acc)] + [(DRAINED, 0)])


@pytest.mark.parametrize("stages,acc", FORMS)
def test_barriers_have_places_of_their_own(place, stages, acc):
    at = [place(stages, acc, *k) for k in kinds(stages, acc)]
    assert sorted(at) == list(range(0, 8 * len(at), 8)) and place(stages, acc, BYTES, 0) == 8 * len(at)


@pytest.mark.parametrize("stages,acc", FORMS)
@pytest.mark.parametrize("tiles", range(6))
@pytest.mark.parametrize("steps", [1, 3, 8])
def test_the_last_wait_is_for_its_own_commit(place, stages, acc, tiles, steps):
    """phases[b]: completed phases of the barrier at byte b, after `tiles` whole tiles and each part of another."""
    for extra in range(steps + 1):
        phases = dict.fromkeys(range(0, place(stages, acc, BYTES, 0), 8), 0)
        it = 0
        for t in range(tiles + 1):
            for step in range(steps if t < tiles else extra):
                phases[place(stages, acc, FULL, it % stages)] += 1
                phases[place(stages, acc, EMPTY, it % stages)] += 1
                it += 1
            if t < tiles:
                phases[place(stages, acc, ACC_FULL, t % acc)] += 1
                phases[place(stages, acc, ACC_EMPTY, t % acc)] += 1
        # a wait for parity 0 returns once an odd number of phases is over
        drained = place(stages, acc, DRAINED, 0)
        assert phases[drained] % 2 == 0
        phases[drained] += 1
        assert phases[drained] % 2 == 1
        # a tile's barrier would not do: after one use its phase of parity 0 is over already
        assert tiles % (2 * acc) != 1 or phases[place(stages, acc, ACC_FULL, 0)] % 2 == 1


def test_both_forms_wait_for_it_whatever_happened():
    """Each form commits on that barrier once and waits for its first phase, under no condition on who gave up."""
    text = (ROOT / "mxfp8-quantizer_b200" / "csrc" / "mxfp4_gemm.cu").read_text()
    assert text.count("mbar_init(drained, 1)") == 2 and text.count("mbar_wait_bounded(drained, 0, kWaitNs)") == 2
    assert text.count("tcgen05_commit<1>(drained)") == 1 and text.count("tcgen05_commit<2>(drained)") == 1
    assert "if (ctl[0])" not in text


def test_each_cta_of_a_pair_waits_for_its_own_arrival():
    """The even CTA's commit arrives in both: a CTA that left without waiting could be gone when it does."""
    text = (ROOT / "mxfp8-quantizer_b200" / "csrc" / "mxfp4_gemm.cu").read_text()
    wide = text[text.index("mxfp4_gemm_wide_kernel("):]
    wait = wide[:wide.index("mbar_wait_bounded(drained, 0, kWaitNs)")]
    last = [line.strip() for line in wait.splitlines() if line.strip()][-2:]
    assert last[0] == "if (warp == kLoadWarp) {" and last[1].startswith("drain_stages<")
