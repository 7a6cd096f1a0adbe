"""``bench.py`` says what it is at, names a kernel wait that ran out and ends when a phase does not."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def run(body, timeout=120):
    return subprocess.run([sys.executable, "-c", f"import sys, time; sys.path.insert(0, {str(ROOT)!r}); import bench\n{body}"],
                          capture_output=True, text=True, timeout=timeout)


def test_a_phase_that_does_not_end_ends_the_process():
    r = run("p = bench.Phases(1.0)\np('warm-up')\np('timed steps')\ntime.sleep(60)")
    assert r.returncode == 1
    assert "] warm-up" in r.stderr and "] timed steps" in r.stderr and "Timeout" in r.stderr and "line 5" in r.stderr


def test_phases_that_end_leave_the_process_alone():
    r = run("p = bench.Phases(1.0, error_word=lambda: 0)\np('warm-up')\np('timed steps')\np.done()\ntime.sleep(2)\nprint('end')")
    assert r.returncode == 0 and r.stdout == "end\n", r.stderr


def test_an_error_word_is_named_with_its_phase():
    r = run("p = bench.Phases(60.0, error_word=lambda: 0x474D)\np('warm-up')\np('timed steps')")
    assert r.returncode == 1 and "0x474d (b'GM') after phase 'warm-up'" in r.stderr and "timed steps" not in r.stderr


def test_an_error_word_that_cannot_be_read_is_an_error():
    r = run("p = bench.Phases(60.0, error_word=lambda: -3)\np('warm-up')\np.done()")
    assert r.returncode == 1 and "cannot be read (code -3) after phase 'warm-up'" in r.stderr
