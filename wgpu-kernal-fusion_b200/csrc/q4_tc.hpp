// Products with 4-bit weights for many rows on the tensor cores (q4_tc.cu)
#pragma once
#include "decode.hpp"

namespace wgf {

struct Q4TcPlan {
    int tile_rows = 0;                 // rows of x of a tile
    int whole = 0;                     // tiles that one CTA does from end to end; the others are done in
    int shares = 1, share_chunks = 0;  // shares of so many steps
    double us = 1e300;                 // about what it takes
};
// parts: 1, or 3 for rows of f32, as three parts of bf16
constexpr int kSplitRows = 32;
Q4TcPlan q4_tc_plan(Device& dev, const Q4Weight& w, int64_t rows, int parts);
// x [rows, k] of 16 bits with a dense last axis and rows `stride` apart, from 16-byte borders on; in three parts: those of 32 rows of f32
// after those of the 32 before, [rows / 32][part][32][k].  y [rows, n], f32 for three parts.
void q4_tc_run(Device& dev, const Q4Weight& w, const Q4TcPlan& plan, const void* x, DType dtype, int64_t stride, int64_t rows, int parts, void* y);

}  // namespace wgf
