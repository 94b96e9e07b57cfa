"""The chunks that the log probability kernel divides a thread's vectors into, by the kernel's own function on the host."""
import pathlib
import re
import shutil
import subprocess

import pytest

SOURCE = pathlib.Path(__file__).resolve().parents[1] / "flex_shard_b200" / "csrc" / "logprobs.cu"


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_chunks_hold_all_vectors_and_shift_by_less_than_a_word(tmp_path):
    text = SOURCE.read_text()
    function = re.search(r"constexpr int chunk_bits\(int n\) \{.*?\n\}", text, re.S)
    most = re.search(r"constexpr int MAX_CHUNKS = \d+;", text)
    assert function and most
    (tmp_path / "c.cpp").write_text(f"#include <cstdio>\n{most[0]}\n{function[0]}\n"
                                    'int main() { for (int n = 0; n < 70000; ++n) std::printf("%d ", chunk_bits(n)); }')
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", str(tmp_path / "c.cpp"), "-o", str(tmp_path / "c")], check=True)
    bits = [int(v) for v in subprocess.run([str(tmp_path / "c")], check=True, capture_output=True, text=True).stdout.split()]
    assert len(bits) == 70000
    for n, b in enumerate(bits):
        assert 2 <= b < 16 and n <= 8 << b and (b == 2 or n > 8 << (b - 1))
