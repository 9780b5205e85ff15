"""How the work of trees of drafts is shared out: the host logic alone, compiled for the CPU."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_sharing_out_ends_and_fits_for_any_sizes(tmp_path):
    exe = str(tmp_path / 'tree_shares_test')
    subprocess.run(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', os.path.join(HERE, 'tree_shares_test.cpp'), '-o', exe], check=True)
    done = subprocess.run([exe], capture_output=True, text=True, timeout=20)
    assert done.returncode == 0, done.stdout[-2000:]
