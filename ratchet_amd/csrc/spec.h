// Host-side rules of the Matmul operator: shape inference, guards, operand
// stacking and the lowering of a descriptor to the strided problem the
// gfx950 kernels consume.  Pure host code: nothing here touches HIP.
#pragma once
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/ratchet_hip.h"

namespace rt {

using Shape = std::vector<int64_t>;

inline bool is_quantized(int dt) { return dt == RT_Q8_0F || dt == RT_Q8_0H || dt == RT_Q4_K || dt == RT_Q4_0; }
inline bool is_float(int dt) { return dt == RT_F32 || dt == RT_F16; }
inline bool valid_dtype(int dt) { return dt >= RT_F32 && dt <= RT_Q4_0; }
// DType::activation_dt (crates/ratchet-core/src/dtype/mod.rs:77-83); Q4_K and Q4_0 pair with f16.
inline int activation_dt(int dt) {
    switch (dt) {
    case RT_Q8_0F: return RT_F32;
    case RT_Q8_0H: return RT_F16;
    case RT_Q4_K:
    case RT_Q4_0: return RT_F16;
    default: return dt;
    }
}
inline int64_t block_numel(int dt) { return dt == RT_Q4_K ? 256 : (is_quantized(dt) ? 32 : 1); }
inline int64_t numel(const Shape &s) {
    int64_t n = 1;
    for (auto d : s) n *= d;
    return n;
}

// Shape::is_vector (crates/ratchet-core/src/shape.rs:71-75).
bool is_vector(const Shape &s);
// Shape::multi_broadcast for two shapes (shape.rs:118-136); false when incompatible.
bool multi_broadcast(const Shape &a, const Shape &b, Shape &out);

// Matmul::compute_c_shape (crates/ratchet-core/src/ops/matmul.rs:284-361).
rt_status compute_c_shape(const Shape &a, const Shape &b, bool trans_lhs, bool trans_rhs, bool trans_out,
                          Shape &out, std::string *why = nullptr);

// The strided problem handed to the kernels.  Operand A is the one that may be
// quantized and is always addressed as rows i of K; operand B supplies the
// columns j.  Element addresses, in elements of the operand's logical dtype:
//   A(s,i,k) = (s % a_stack) * a_bs + i * a_rs + k * a_ks
//   B(s,k,j) = (s % b_stack) * b_bs + k * b_ks + j * b_js
//   O(s,i,j) =  s * o_bs            + i * o_is + j * o_js
struct Problem {
    int a_dt = RT_F32;   // storage dtype of A (may be quantized)
    int act_dt = RT_F32; // dtype of B, bias and the output
    int64_t stacks = 1, a_stack = 1, b_stack = 1;
    int64_t M = 0, N = 0, K = 0; // rows of A, columns of B, contraction
    int64_t a_bs = 0, a_rs = 0, a_ks = 0;
    int64_t b_bs = 0, b_ks = 0, b_js = 0;
    int64_t o_bs = 0, o_is = 0, o_js = 0;
    bool has_bias = false;
    bool bias_on_rows = false; // bias indexed by i (rows of A) rather than by j
    bool swapped = false;      // A is the descriptor's rhs
    int act = 0;               // rt_activation applied to (product + bias) before the output is rounded
    int kernel = RT_KERNEL_NONE;
    // caller-provided device memory a launcher may use to share one problem's K among workgroups
    void *workspace = nullptr;
    uint64_t workspace_bytes = 0;
};

// Limits of the streaming (GEMV) kernels: number of activation vectors.
constexpr int kGemvMaxCols = 8;      // VALU kernels (f16/f32/Q8_0F weights)
constexpr int kGemvQ8hMaxCols = 16;  // matrix-core kernel (Q8_0H weights)
constexpr int kGemvQ4kMaxCols = 16;  // matrix-core kernel (Q4_K weights); the VALU one takes up to kGemvMaxCols
constexpr int kGemvQ40MaxCols = 64;  // matrix-core kernel (Q4_0 weights)

rt_status validate(const rt_matmul_desc &d, std::string *why = nullptr);
rt_status infer(const rt_matmul_desc &d, Shape &out, int &out_dt, std::string *why = nullptr);
rt_status make_spec(const rt_matmul_desc &d, rt_gemm_spec &spec, Problem &prob, std::string *why = nullptr);

} // namespace rt
