"""The numbers of decode attention's rounds, tags of the words that its CTAs exchange
(csrc/attn_tags.h): none is met twice, however long a process decodes."""
import os
import subprocess

from conftest import PKG_DIR

HERE = os.path.dirname(os.path.abspath(__file__))


def test_no_word_passes_as_a_later_rounds(tmp_path):
    exe = str(tmp_path / "attn_tags_test")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror",
                    "-I", os.path.join(PKG_DIR, "csrc"),
                    os.path.join(HERE, "fake_cuda", "attn_tags_test.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
