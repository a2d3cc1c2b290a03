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
// exact: rows of f32, as three parts of bf16
constexpr int kExactRows = 32;
Q4TcPlan q4_tc_plan(Device& dev, const Q4Weight& w, int64_t rows, bool exact);
// x [rows, k] of 16 bits with a dense last axis and rows `stride` apart, from 16-byte borders on; exact: the parts of 32 rows of f32
// after those of the 32 before, [rows / 32][part][32][k].  y [rows, n], f32 if exact.  False where x cannot be brought by TMA.
bool q4_tc_run(Device& dev, const Q4Weight& w, const Q4TcPlan& plan, const void* x, DType dtype, int64_t stride, int64_t rows, bool exact, void* y);

}  // namespace wgf
