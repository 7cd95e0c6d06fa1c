"""An error whose message holds a number raises; it must not end the process (run in one of its own)."""
import subprocess
import sys

from conftest import ROOT


def test_a_number_in_an_error_message_raises(built_libs):
    code = ("import cuda_agent_b200\next = cuda_agent_b200.load_extension()\n"
            "try:\n    ext.moe_ep_status(12345)\nexcept RuntimeError as e:\n    assert '12345' in str(e), e\n    print('raised')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "raised" in run.stdout, (run.returncode, run.stderr)
