"""Where the 8-bit product's tiles load (slam_amd/csrc/gemm_fp8_plan.h, compiled for the host): every access that an operand's range check
lets through lies inside the operand, whether or not the check counts the scalar offset, and every element that a tile needs is loaded."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slam_amd", "csrc")
SOURCE = """
#include "gemm_fp8_plan.h"
using namespace slamhip;
extern "C" {
// vector and scalar offsets of the loads of `rows_on` rows behind rows first .. first + 7, blocks 0 .. blocks - 1, chunks 0 .. 7
void operand(int first, int rows_on, int blocks, int K, unsigned* vec, unsigned* sca) {
  for (int r = 0; r < 8; ++r)
    for (int kb = 0; kb < blocks; ++kb)
      for (int c = 0; c < 8; ++c, ++vec, ++sca) {
        *vec = operand_load(operand_offset(first + r, c, K), kb, c, rows_on, K);
        *sca = block_offset(kb, (K + 127) / 128);
      }
}
void scale(int row0, int rows_in_tile, int blocks, int rows, int KB, unsigned* vec) {
  for (int r = 0; r < rows_in_tile; ++r)
    for (int kb = 0; kb < blocks; ++kb) *vec++ = scale_load(row0 + r, kb, rows, KB);
}
void plan(int M, int N, int K, long long* out) {
  const GemmPlan g = gemm_plan(M, N, K);
  out[0] = g.kind, out[1] = g.groups, out[2] = g.per, out[3] = g.parts;
}
}
"""
KINDS = ("rows", "256x256", "128x128", "128x128 KW", "64x128 KW", "64x64 KW")
# rows of a tile (of the first operand, of the second) and waves that load one slice
TILES = {"256x256": (256, 256, 8), "128x128": (128, 128, 4), "128x128 KW": (128, 128, 4), "64x128 KW": (64, 128, 4), "64x64 KW": (64, 64, 4)}
AHEAD = 9     # blocks behind the last that the loops ask for: four slices of two groups, and one


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-Wno-unused-function", "-fPIC", "-shared", "-I" + CSRC, "-o", str(d / "plan.so"),
                           str(d / "plan.cpp")])
    return ctypes.CDLL(str(d / "plan.so"))


def plan(lib, M, N, K):
    out = (ctypes.c_longlong * 4)()
    lib.plan(M, N, K, out)
    return KINDS[out[0]], out[1], out[2], out[3]


def operand_loads(lib, rows, K, tile_rows, waves, former=False):
    """(row, block, chunk, vector offset, scalar offset) of all loads of all tiles over an operand of `rows` rows."""
    KB = -(-K // 128)
    blocks = KB + AHEAD
    parts = []
    for first in range(0, -(-rows // tile_rows) * tile_rows, tile_rows):
        for wave in range(waves):
            for i in range(tile_rows // 8 // waves):
                row = first + wave * 8
                shape = (8, blocks, 8)
                vec, sca = np.empty(shape, np.uint32), np.empty(shape, np.uint32)
                r, kb, c = np.meshgrid(np.arange(8), np.arange(blocks), np.arange(8), indexing="ij")
                if former:      # the group of rows in the scalar offset
                    vec[:] = np.where(kb * 128 + c * 16 < K, (row + r) * K + c * 16, 0x80000000)
                    sca[:] = kb * 128 + i * waves * 8 * K
                else:
                    lib.operand(row, i * waves * 8, blocks, K, vec.ctypes.data_as(ctypes.c_void_p), sca.ctypes.data_as(ctypes.c_void_p))
                parts.append([v.ravel().astype(np.int64) for v in (row + i * waves * 8 + r, kb, c, vec, sca)])
    return [np.concatenate(v) for v in zip(*parts)]


def outside(vec, sca, size, width, counted):
    """Accesses that pass the range check and touch what is behind the operand."""
    through = vec < size - sca if counted else vec < size
    if counted:
        through |= size < sca           # a difference of unsigned numbers
    return through & (vec + sca + width > size)


# operands with short edges of every kind: fewer rows than a tile and than a group of rows, one row over, K below and behind a block's end
SHAPES = [(1, 16), (17, 16), (17, 4096), (33, 144), (63, 128), (64, 400), (65, 272), (130, 640), (192, 2064), (200, 128), (255, 48), (256, 256), (257, 1040),
          (300, 2048), (513, 144)]


@pytest.mark.parametrize("kind", sorted(TILES))
@pytest.mark.parametrize("rows,K", SHAPES)
def test_loads_stay_inside_the_operands(lib, kind, rows, K):
    bm, bn, waves = TILES[kind]
    for tile_rows in {bm, bn}:
        row, kb, c, vec, sca = operand_loads(lib, rows, K, tile_rows, waves)
        size = rows * K
        assert (vec + sca < 1 << 32).all()
        for counted in (False, True):
            assert not outside(vec, sca, size, 16, counted).any(), (tile_rows, counted)
        # what belongs to the operand comes from its place, all else from behind it
        own = (row < rows) & (kb * 128 + c * 16 < K)
        assert np.array_equal((vec + sca)[own], (row * K + kb * 128 + c * 16)[own])
        assert (vec[~own] >= size).all()


@pytest.mark.parametrize("kind", sorted(TILES))
def test_the_check_sees_a_row_in_the_scalar_offset(lib, kind):
    """With the group of rows in the scalar offset, as it was, a range check of the vector offset alone lets reads behind the operand through."""
    bm, bn, waves = TILES[kind]
    _, _, _, vec, sca = operand_loads(lib, 17, 4096, bn, waves, former=True)
    assert outside(vec, sca, 17 * 4096, 16, counted=False).any()


@pytest.mark.parametrize("rows,KB", [(17, 1), (17, 3), (64, 4), (65, 5), (255, 32), (257, 7), (300, 1)])
def test_scale_loads_stay_inside(lib, rows, KB):
    for bm in (64, 128, 256):
        blocks = (KB + 3) // 4 * 4 + 12
        for row0 in range(0, rows, bm):
            vec = np.empty((bm, blocks), np.uint32)
            lib.scale(row0, bm, blocks, rows, KB, vec.ctypes.data_as(ctypes.c_void_p))
            r, kb = np.meshgrid(row0 + np.arange(bm), np.arange(blocks), indexing="ij")
            own = (r < rows) & (kb < KB)
            assert np.array_equal(vec[own], (r * KB + kb)[own] * 4)
            assert (vec[~own] >= rows * KB * 4).all()


def test_offsets_of_the_largest_operands(lib):
    """(rows + 256) K just below 2^31: offsets behind the operand do not come round to its beginning."""
    vec, sca = np.empty((8, 9, 8), np.uint32), np.empty((8, 9, 8), np.uint32)
    at = lambda v: v.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    for rows, K in ((16, 7895152), ((1 << 27) - 257, 16), (523000, 4096), (7743, 268432)):
        assert (rows + 256) * K < 1 << 31
        for first, on in ((rows // 256 * 256, 248), (rows - 8, 0), (rows // 256 * 256 + 56, 192)):
            lib.operand(first, on, 9, K, at(vec), at(sca))
            row = first + on + np.arange(8)
            v = vec.astype(np.int64)
            assert (v[row >= rows] >= rows * K).all() and (v + sca < 1 << 32).all()


def test_the_plan_covers_every_tile(lib):
    for M, N, K in ((1, 1, 16), (16, 4096, 4096), (17, 64, 16), (777, 2056, 4096), (5000, 4096, 4096), (100, 500, 16384), (5, 40, 8336)):
        kind, groups, per, parts = plan(lib, M, N, K)
        KB = -(-K // 128)
        bm, bn = (16, 16) if kind == "rows" else TILES[kind][:2]
        assert groups == (1 if kind == "rows" else -(-M // bm)) * -(-N // bn)
        assert per % 4 == 0 and parts * per >= KB > (parts - 1) * per


def test_the_long_products_reach_every_kind(lib):
    """The shapes that the GPU tests take for each kind: one part of k, more blocks than the buffers of slices and of scales hold."""
    from test_sequence_ops_long_gpu import GEMM_LONG
    assert sorted(GEMM_LONG) == sorted(KINDS)
    for kind, (M, N, K) in GEMM_LONG.items():
        got, _, per, parts = plan(lib, M, N, K)
        assert got == kind and parts == 1 and per >= 18 and K % 128, kind
