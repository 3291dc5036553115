"""The scratch of a head's gradients: what each launch of each piece of the classes writes lies in the part that it is given. The
plan is host arithmetic (csrc/loss_plan.h), compiled here by itself and gone through over sizes and numbers of SMs."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnabla_b200", "csrc")

PROGRAM = r"""
#include "loss_plan.h"
using namespace nb200;
// out: for G, dx's sums, dW's sums and db's sums the room and, over all pieces, the end of what is written, in bytes;
// then the rows of G that db's sums leave out
extern "C" void plan(int64_t rows, int64_t size, int64_t classes, int f32, int accum_dx, int64_t x_bytes, int64_t w_bytes,
                     int sms, int64_t *out) {
  const HeadGradients p(rows, size, classes, f32, true, true, true, accum_dx, x_bytes, w_bytes, sms);
  const size_t at[5] = {p.at_g, p.at_dx, p.at_dw, p.at_db, p.bytes};
  out[0] = p.at_scale - p.at_g;
  for (int i = 1; i < 4; ++i)
    out[2 * i] = at[i + 1] - at[i];
  out[1] = out[3] = out[5] = out[7] = out[8] = 0;
  for (int64_t c0 = 0; c0 < classes; c0 += p.piece) {
    const int64_t n = p.classes_at(c0);
    auto most = [&](int i, int64_t v) { out[i] = std::max(out[i], v); };
    // G: whole chunks of 32 classes of each row
    most(1, ((p.planes * rows - 1) * p.piece + up(n, 32)) * 2);
    if (!p.direct)
      most(3, (((n + 63) / 64 + p.dx_blocks - 1) / p.dx_blocks * rows - 1) * p.ld_dx * 4 + size * 4);
    if (p.dw_splits > 1)
      most(5, ((p.dw_splits * size - 1) * p.piece + n) * 4);
    const Slabs s = p.db; // (a block writes its 256 sums up to the pitch)
    most(7, ((s.count - 1) * p.piece + std::min(p.piece, up(n, kSumColumns))) * 4);
    most(8, std::max<int64_t>(0, p.planes * rows - s.count * s.rows));
  }
}
"""


PROGRAM += r"""
extern "C" void few(int64_t size, int64_t classes, int vec, int shift, int sms, int64_t *out) {
  const FewGradients p(size, classes, vec, shift, sms);
  out[0] = p.columns, out[1] = p.slab, out[2] = p.blocks;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cc, "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + CSRC, str(d / "plan.cpp"), "-o", str(d / "plan.so")],
                   check=True)
    return ctypes.CDLL(str(d / "plan.so"))


@pytest.fixture(scope="module")
def plan(lib):
    def f(rows, size, classes, f32, accum=False, sms=148):
        out = (ctypes.c_int64 * 9)()
        i = ctypes.c_int64
        pitch = (classes + 63) // 64 * 64
        lib.plan(i(rows), i(size), i(classes), int(f32), int(accum), i(3 * rows * size * 2), i(size * pitch * 6), sms, out)
        return list(out)
    return f


def inside(out):
    rooms, written = out[0:8:2], out[1:8:2]
    return all(w <= r for r, w in zip(rooms, written)) and out[8] == 0


@pytest.mark.parametrize("rows,classes,f32", [(8192, 128000, False), (4096, 50257, False), (1024, 50257, False), (4096, 50257, True),
                                              (2048, 20011, False), (2048, 20011, True), (8192, 128000, True),
                                              (20000, 32700, False), (256, 1000, True), (1000, 10007, True)])
@pytest.mark.parametrize("sms", [148, 132, 64, 2])
def test_a_last_piece_with_fewer_classes(plan, rows, classes, f32, sms):
    for size in (16, 777, 2048):
        out = plan(rows, size, classes, f32, sms=sms)
        assert inside(out), out


def test_sizes_at_random(plan):
    rng = random.Random(5)
    spread = lambda a, b: int(round(a * (b / a) ** rng.random()))
    for _ in range(20000):
        rows, size, classes = spread(9, 1 << 20), spread(1, 20000), spread(1, 1 << 20)
        args = (rows, size, classes, rng.random() < 0.5, rng.random() < 0.3, rng.choice([148, 148, 132, 80, 20, 2]))
        out = plan(*args)
        assert inside(out), (args, out)


def test_blocks_of_few_rows_cover_the_weights(lib):
    """Every row of W once, in blocks of rows that lie `vec` apart where they begin anywhere, and every class; in a grid's limits."""
    rng = random.Random(6)
    spread = lambda a, b: int(round(a * (b / a) ** rng.random()))
    for _ in range(5000):
        size, classes, vec = spread(1, 1 << 24), spread(1, (1 << 24) - 1), rng.choice([4, 8])
        shift = rng.random() < 0.5 or classes % vec != 0
        out = (ctypes.c_int64 * 3)()
        lib.few(ctypes.c_int64(size), ctypes.c_int64(classes), vec, int(shift), rng.choice([148, 132, 2]), out)
        columns, slab, blocks = out
        step = vec if shift else 1
        assert slab % 32 == 0 and blocks % step == 0 and blocks <= 65535 and columns < 1 << 31
        assert blocks // step * slab >= -(-size // step) > (blocks // step - 1) * slab
        # (the rows' ends have a block column of their own)
        assert 2048 * (columns - (1 if shift else 0)) >= classes + (vec - 1 if shift else 0)
