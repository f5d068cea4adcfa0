"""The linear operator's steps and pieces of a row, up to the longest row that its entry accepts (2^31 - 2 bytes),
compiled for the host and compared with 64-bit arithmetic under the checks for undefined behaviour."""
import subprocess

from sparsesnn_amd import build

SOURCE = r"""
#include <cstdio>
#include "sparsesnn_amd/csrc/linear.h"
int main() {
  const int rows[] = {0, 1, 15, 16, 17, 127, 128, 129, 1 << 20, 0x3fffffff, 0x7fffff7f, 0x7fffff80, 0x7fffff81,
                      0x7fffffef, 0x7ffffff0, 0x7ffffff1, 0x7ffffffe, 0x7fffffff};
  for (const int kb : rows) {
    const long long steps = ((long long)kb + 127) / 128, first = steps > 3 ? steps - 3 : 0;
    long long n = first;
    for (uint32_t k = (uint32_t)(first * 128); sengine::has_step(k, kb); k = sengine::next_step(k), ++n) {
      if (n >= steps || k != n * 128) return std::printf("step %lld of %d bytes\n", n, kb), 1;
      for (int at = 0; at < 128; at += 16) {
        const long long left = (long long)kb - (n * 128 + at);
        if (left > 0 && sengine::whole_piece((int)k + at, kb) != (left >= 16))
          return std::printf("piece at %d of step %lld of %d bytes\n", at, n, kb), 1;
      }
    }
    if (n != steps) return std::printf("%lld steps of %d bytes\n", n, kb), 1;
  }
  return 0;
}
"""


def test_steps_and_pieces(tmp_path):
    src, exe = tmp_path / "steps.hip", tmp_path / "steps"
    src.write_text(SOURCE)
    flags = [f for f in build.HIPCC_FLAGS if f != "-O3"]
    subprocess.run([build.hipcc(), *flags, "--offload-host-only", "-Xarch_host", "-fsanitize=undefined", "-Xarch_host",
                    "-fno-sanitize-recover=all", str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
