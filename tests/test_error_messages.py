"""An error whose message holds a number raises; it must not end the process (run in one of its own)."""
import subprocess
import sys

from conftest import ROOT


def test_a_number_in_an_error_message_raises(built_libs):
    code = ("import cuda_agent_b200\next = cuda_agent_b200.load_extension()\n"
            "try:\n    ext.moe_ep_status(12345)\nexcept RuntimeError as e:\n    assert '12345' in str(e), e\n    print('raised')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "raised" in run.stdout, (run.returncode, run.stderr)


def test_the_extension_links_with_compilers_that_have_fewer_options(built_libs, tmp_path, monkeypatch):
    """g++ knows -nostdlib++ from version 13 on; one that does not has to link the same module, on the shared C++ runtime."""
    old = tmp_path / "g++"
    old.write_text('#!/bin/sh\nfor a in "$@"; do if [ "$a" = "-nostdlib++" ]; then echo "unrecognized option $a" >&2; exit 1; fi; done\n'
                   f'exec "{built_libs.CXX}" "$@"\n')
    old.chmod(0o755)
    monkeypatch.setattr(built_libs, "CXX", str(old))
    monkeypatch.setattr(built_libs, "EXT_SO", tmp_path / "cuda_extension.so")
    monkeypatch.setattr(built_libs, "_compile_one", lambda src, compiler, flags: (built_libs.OBJ_DIR / (src.name + ".o"), False))
    needed = subprocess.run(["readelf", "-d", str(built_libs.build_extension())], capture_output=True, text=True, check=True).stdout
    assert "[libstdc++.so.6]" in needed
