// The digit tables of SoftmaxLastAxis at the model scale S = 2^14 (atlas-onnx-tracer/src/ops/softmax.rs:239-269) as compile-time constants:
// exp(-z / S) S ~ HI[z >> 9] LO[z & 511] / S with HI[h] = round(S exp(-512 h / S)), LO[l] = round(S exp(-l / S)).  The graph executor builds the
// same numbers at run time and uploads them (graph_exec.hip: atlas_rt_exp_lut); as constants of the code object they need no upload, so
// the first call of an attention entry point may already be inside a stream capture.  tests/test_attention.py compares the two.
#pragma once
#include <cstdint>

namespace atlas {
struct ExpTable {
    static constexpr int LOG_BASE = 9, BASE = 1 << LOG_BASE, HI = 512, HI_USED = 334, Z_MAX = HI * BASE - 1;
    int32_t hi[HI], lo[BASE];
};
// exp(-x), 0 <= x < 16: the series at x / 2^6 (|term| < 2^-60 after 24 of them), squared six times; the relative error stays below 2^-44, the
// nearest any entry comes to a rounding border is far above that
constexpr double exp_neg(double x) {
    const double y = -x / 64.0;
    double term = 1.0, sum = 1.0;
    for (int i = 1; i <= 24; i++) { term *= y / i; sum += term; }
    for (int i = 0; i < 6; i++) sum *= sum;
    return sum;
}
constexpr ExpTable make_exp_table() {
    ExpTable t{};
    for (int h = 0; h < ExpTable::HI; h++) t.hi[h] = h < ExpTable::HI_USED ? (int32_t)(16384.0 * exp_neg(h / 32.0) + 0.5) : 0;
    for (int l = 0; l < ExpTable::BASE; l++) t.lo[l] = (int32_t)(16384.0 * exp_neg(l / 16384.0) + 0.5);
    return t;
}
}  // namespace atlas
