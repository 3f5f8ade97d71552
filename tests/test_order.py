"""The order in which a run of all tests takes them."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))


def test_tests_that_pass_made_up_addresses_run_before_the_library_is_initialised():
    run = subprocess.run([sys.executable, "-m", "pytest", "--collect-only", "-q", "tests/test_gpu_kv4_refusals.py",
                          "tests/test_abi.py", "tests/test_gpu_kv4_rows.py", "tests/test_kv4.py"],
                         cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=110)
    files = [line.split("::")[0] for line in run.stdout.splitlines() if "::" in line]
    gpu = ["test_gpu" in f for f in files]
    assert gpu.count(True) > 5 and gpu.count(False) > 50 and gpu == sorted(gpu), run.stdout[-500:]
