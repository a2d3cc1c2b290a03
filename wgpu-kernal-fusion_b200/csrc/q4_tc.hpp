// Products with 4-bit weights for many rows of 16-bit types (q4_tc.cu)
#pragma once
#include "decode.hpp"

namespace wgf {

struct Q4TcPlan {
    int tile_rows = 0;                 // rows of x of a tile
    int whole = 0;                     // tiles that one CTA does from end to end; the others are done in
    int shares = 1, share_chunks = 0;  // shares of so many steps
    double us = 1e300;                 // about what it takes
};
Q4TcPlan q4_tc_plan(Device& dev, const Q4Weight& w, int64_t rows);
// x [rows, k] with a dense last axis, rows from 16-byte borders on; y [rows, n].  False where x cannot be brought by TMA.
bool q4_tc_run(Device& dev, const Q4Weight& w, const Q4TcPlan& plan, const TensorData& x, int64_t rows, void* y);

}  // namespace wgf
