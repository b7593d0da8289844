"""The Node-API shim's checks of the paged cache's and qkNormRope's arguments, from JavaScript; the library is not reached."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_arguments_that_are_no_ids_lengths_or_numbers_throw():
    node = shutil.which("node")
    if node is None:
        pytest.skip("no node binary on this machine")
    if not os.path.exists(os.path.join(ROOT, "framework_amd", "lib", "mni_rocm.node")):
        pytest.skip("Node addon not built (node_api.h missing at build time)")
    p = subprocess.run([node, os.path.join(ROOT, "tests", "js", "paged_arguments.js")], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and " 0 failed" in p.stdout, p.stdout + p.stderr
