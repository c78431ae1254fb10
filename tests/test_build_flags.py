"""What the kernels are compiled with, checked on a kernel that invites it."""
import subprocess

from video_rep_learning_amd.csrc import build

SOURCE = """
#include <hip/hip_runtime.h>
typedef float f2 __attribute__((ext_vector_type(2)));
extern "C" __global__ void pairs(f2* x, const f2* y) {
  const f2 a = x[threadIdx.x], b = y[threadIdx.x];
  x[threadIdx.x] = __builtin_elementwise_fma(a, b, a * a) + b;
}
"""


def assembly(flags, tmp_path):
    src, out = tmp_path / 'pairs.hip', tmp_path / 'pairs.s'
    src.write_text(SOURCE)
    r = subprocess.run([build.HIPCC] + flags + ['--cuda-device-only', '-S', str(src), '-o', str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out.read_text()


def test_no_packed_fp32_instructions(tmp_path):
    """Every source is compiled with the same flags, and they make none (without them this kernel has some)."""
    assert 'v_pk_' not in assembly(build.FLAGS, tmp_path)
    at = build.FLAGS.index('-packed-fp32-ops')
    assert build.FLAGS[at - 3:at] == ['-Xclang', '-target-feature', '-Xclang']
    assert 'v_pk_' in assembly(build.FLAGS[:at - 3] + build.FLAGS[at + 1:], tmp_path)
