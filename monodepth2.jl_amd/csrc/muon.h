// muon.h -- host interface of muon.hip (Newton-Schulz orthogonalisation, its pullback, the Muon update)
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#define MD2_NS_MAX_STEPS 16

namespace md2 {

enum { NS_F32 = 0, NS_BF16 = 1, NS_F16 = 2 };                     // element types of the caller's matrices
enum { NS_FORWARD = 0, NS_BACKWARD = 1, NS_MUON = 2 };

// one weight, or a batch of equal matrices; strides in elements (batch, row, column)
struct NsMatrices {
    const void* x = nullptr; const void* d = nullptr; void* y = nullptr;      // forward: matrix, -, result | backward: matrix, dout, dx | Muon: momentum (updated), gradient, weight (updated)
    int64_t batch = 1, rows = 0, cols = 0, xs[3] = {0, 0, 0}, ds[3] = {0, 0, 0};
    float alpha = 0.f;                                            // Muon: learning rate * shape factor
};
struct NsOptions {
    int steps = 5; double coef[3] = {3.4445, -4.7750, 2.0315}, eps = 1e-7;
    double lr = 0, momentum = 0, weight_decay = 0; int nesterov = 1; float grad_scale = 1.f;
};
// why these are refused, or null
const char* ns_check(int steps, const double* coefficients, double eps);
// bytes of workspace, -1 for sizes that are refused
int64_t ns_workspace(int kind, int steps, const NsMatrices* q, int count);
// which kernels a call takes: tile side and pieces of the K axis of X X^T, b A + c A A, S, V and (pieces 1) the products with m x n; sides 0: none such, or the call is one launch.  -1 for sizes
// that are refused
int ns_tiles(int kind, int steps, const NsMatrices* q, int count, int32_t side[5], int32_t pieces[5]);
// enqueues on s; 0, or 2 with the reason in *why (nothing was enqueued)
int ns_run(int kind, int dtype, const NsMatrices* q, int count, const NsOptions& o, void* ws, int64_t ws_bytes, hipStream_t s, const char** why);

}  // namespace md2
