// Parameters and launchers of the sequence operators: layer norm, the short causal convolution and the selective state
// space scan on tensors of rows, [sequences][tokens][channels].
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200conv.h"

namespace b200 {

inline size_t row_elem_size(int dtype) { return dtype == B200CONV_F32 ? 4 : 2; }

// 16-byte accesses to every row of a tensor: what the vector forms of the kernels ask for.
inline bool rows_aligned(const void* p, const b200conv_rows& r, int dtype) {
  const long long es = static_cast<long long>(row_elem_size(dtype));
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && !(r.row * es % 16) && !(r.seq * es % 16));
}

// ---- layer norm (layer_norm.cu) ----
struct NormArgs {
  b200conv_norm_desc d;
  const void *x, *residual, *gamma, *beta, *dy, *dtotal;
  void *y, *total, *dx, *dgamma, *dbeta;
  float* stats;
  float* partial;          // gradients: [norm_grad_parts][2][C]
};
cudaError_t launch_layer_norm(const NormArgs& a, cudaStream_t s);
int norm_grad_parts(const b200conv_norm_desc& d);
cudaError_t launch_layer_norm_grad(const NormArgs& a, int* launches, cudaStream_t s);

// ---- short causal convolution (causal_conv.cu, causal_conv_grad.cu) ----
struct CausalArgs {
  b200conv_causal_desc d;
  const void *x, *w, *bias, *initial, *dy;
  const int* starts;
  void *y, *final, *dx, *dw, *dbias, *dinitial;
  float* partial;          // gradients: [causal_grad_parts][taps + 1][C]
};
cudaError_t launch_causal_conv(const CausalArgs& a, cudaStream_t s);
cudaError_t launch_causal_step(const CausalArgs& a, cudaStream_t s);
int causal_grad_parts(const CausalArgs& a);
cudaError_t launch_causal_grad(const CausalArgs& a, int* launches, cudaStream_t s);

// ---- selective scan (selective_scan.cu, selective_scan_grad.cu) ----
struct ScanArgs {
  b200conv_scan_desc d;
  const void *x, *dt, *z, *B, *C, *dy;
  const float *A, *D, *dt_bias, *initial, *dfinal;
  const int* starts;
  void *y, *dx, *ddt, *dz, *dB, *dC;
  float *final, *dA, *dD, *ddt_bias, *dinitial;
  // the cut into pieces: tokens of a piece, pieces of a sequence (not of packed ones), of the call; blocks side by side
  int piece, pieces_per_seq, pieces, tiles;
  float *piece_state, *piece_sum;          // [pieces][C][scan_state_slots(N)], [pieces][C]: what a piece makes of zero states, its sum of deltas
  // gradients: rows of the tensors, the states in front of every fourth token ([scan_kept][scan_grad_slots(N) / 4][C] of four) with the sums
  // of deltas up to there, what a piece makes of a zero adjoint, partial sums: [blocks of a group][rows][groups][2][N], [pieces][C][N], [pieces][2][C]
  long long rows;
  float *kept, *kept_sum, *piece_back, *partial_bc, *partial_a, *partial_d;
};
void cut_pieces(ScanArgs* a, long long tiles, long long slots);
void plan_scan_pieces(ScanArgs* a);
int scan_state_slots(int N);               // states of a channel as the workspaces hold them
cudaError_t launch_selective_scan(const ScanArgs& a, int* launches, cudaStream_t s);
void plan_grad_pieces(ScanArgs* a);
int scan_grad_slots(int N);              // the same in those of the gradient
long long scan_kept(const ScanArgs& a);    // kept states per channel
cudaError_t launch_scan_grad(const ScanArgs& a, int* launches, cudaStream_t s);
cudaError_t launch_scan_step(const ScanArgs& a, int* launches, cudaStream_t s);

}  // namespace b200
