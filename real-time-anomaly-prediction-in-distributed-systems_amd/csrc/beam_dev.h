// beam_dev.h -- row moves shared by beam.hip and engine.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/htm_amd.h"

// Buffers of rows: row r of dst[k] becomes a row of src[k], `bytes` each.
struct RowMoves {
    const uint8_t* src[HTM_BEAM_BUFFERS];
    uint8_t* dst[HTM_BEAM_BUFFERS];
    uint64_t bytes[HTM_BEAM_BUFFERS];
    int32_t n;
};

// n_beams > 0: row (g, w) from row (g, idx[g][w]) of its group, in place where
// src == dst; n_beams == 0: row r from row idx[r] of n_src (src != dst)
int rows_move(const RowMoves& m, const int32_t* idx, int64_t n_rows, int32_t n_beams, int64_t n_src, hipStream_t st);
