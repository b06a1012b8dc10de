"""What sd3_linear_residual refuses before any CUDA call, and the rule that picks its kernel (no GPU needed)."""
import os
import subprocess
from ctypes import c_void_p

import pytest

from conftest import REPO, load_binding

P, Q, R = c_void_p(4096), c_void_p(1 << 20), c_void_p(1 << 24)  # never read: every call here is refused


def call(s, x=P, ldx=64, w=Q, ldw=64, bias=None, act=0, residual=None, ldr=0, out=R, ldo=32, dtype=1, M=4, N=32, K=64):
    return s.lib().sd3_linear_residual(x, ldx, w, ldw, bias, act, residual, ldr, out, ldo, dtype, M, N, K, None)


@pytest.mark.parametrize("bad,code", [(dict(dtype=2), -1), (dict(act=5), -1), (dict(act=-1), -1), (dict(M=-1), -1), (dict(N=0), -1),
                                      (dict(K=0), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(out=None), -1), (dict(ldx=56), -1),
                                      (dict(ldw=56), -1), (dict(ldo=31), -1), (dict(residual=R, ldr=31), -1),
                                      (dict(residual=R, ldr=40), -1), (dict(out=c_void_p(4097)), -1), (dict(bias=c_void_p(4098)), -1),
                                      (dict(ldx=65), -2), (dict(ldw=65), -2), (dict(x=c_void_p(4104)), -2), (dict(w=c_void_p(4104)), -2)])
def test_refusals(bad, code):
    s = load_binding()
    assert call(s, **bad) == code
    assert b"sd3_linear_residual" in s.lib().sd3_last_error()


def test_no_rows_need_nothing():
    assert call(load_binding(), x=None, M=0) == 0


def test_plan(tmp_path):
    """Every plan can be launched: a split has K blocks for each of its CTAs and tiles that fit shared memory."""
    src = tmp_path / "plan.cpp"
    src.write_text('''
#include "launch_rules.h"
#include <cstdio>
int main() {
  const int sizes[] = {1, 2, 7, 8, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700, 1536, 4096, 16384, 100000};
  for (int M : sizes) for (int N : sizes) for (int K : sizes) for (int f32 = 0; f32 < 2; ++f32) {
    const int kb = (K + 63) / 64;
    const sd3::LinearPlan p = sd3::linear_plan(M, N, kb, f32 != 0, 148);
    if (p.pair) { if (M <= 128) return 1; continue; }
    if ((p.bn != 64 && p.bn != 128) || p.split < 1 || p.split > 8 || p.split > kb) return 2;
    const int cols = (p.bn / 4 + p.split - 1) / p.split * 4, a_rows = M < 128 ? (M + 7) / 8 * 8 : 128;
    if (cols * p.split < p.bn) return 3;
    int partial = p.split * a_rows * (cols + 4) * 4;
    if (partial < 16384) partial = 16384;  // what an MMA may read behind the last stage
    const int room = 227 * 1024 - 1024 - 208 - partial;
    if (room / (2 * (p.bn + a_rows) * 128) < 2) return 4;  // two stages of two K blocks at least
  }
  std::puts("ok");
}
''')
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(REPO, "sd3.c_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "ok\n"
