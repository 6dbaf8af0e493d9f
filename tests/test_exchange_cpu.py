"""How the CTAs of a cluster leave the exchange of their parts' sums, with threads in the CTAs' place."""
import ctypes
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    out = tmp_path_factory.mktemp("exchange") / "libprobe.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-pthread", "-o", str(out),
                    str(ROOT / "tests" / "cpp" / "exchange_probe.cc")], check=True)
    return ctypes.CDLL(str(out)).probe_exchange


def run(probe, delays, flight, limit):
    late, barriers = ctypes.c_int(), ctypes.c_int()
    wrong = probe(len(delays), (ctypes.c_int * len(delays))(*delays), flight, limit, ctypes.byref(late), ctypes.byref(barriers))
    return wrong, late.value, barriers.value


@pytest.mark.parametrize("delays", [(400, 0), (0, 400, 0, 0), (0, 0, 0, 300, 0, 500, 0, 0)])
def test_no_copy_finds_a_cta_gone_whose_wait_ran_out(probe, delays):
    """Peers that send long after the others' waits ran out: their copies are under way when they reach the barrier."""
    wrong, late, barriers = run(probe, delays, flight=100, limit=50)
    assert late >= len(delays) - 1 and wrong == 0 and barriers == 2


def test_one_barrier_where_everything_came(probe):
    wrong, late, barriers = run(probe, (0, 20, 0, 10), flight=1, limit=20000)
    assert (wrong, late, barriers) == (0, 0, 1)
