"""How the attention's work is shared and joined, without a GPU (under sanitizers), and a refusal of the entry point."""

import os
import shutil
import subprocess

import pytest

from qwenny_amd._lib import KvC, TreeC, lib

HERE = os.path.dirname(os.path.abspath(__file__))
FAKE = 0x10000


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_parts_under_sanitizers(tmp_path):
    exe = str(tmp_path / "driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(HERE, "attn_parts_driver.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_caches_past_32_bit_tiles_are_refused():
    kv = KvC(fmt=1, heads=128, head_dim=64, page=64, pages=(1 << 25) - 1, codes=FAKE, scales=FAKE)
    step = TreeC(n=1, n_seq=1, max_new=1, start=FAKE, len=FAKE, table=FAKE, table_ld=4, mask=None)
    assert lib().qh_tree_attn(None, None, FAKE, 128, kv, step, 0.1, None, FAKE) == -1
    assert "too large" in lib().qh_last_error().decode()
