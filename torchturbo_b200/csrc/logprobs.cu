// Log-probabilities of rows of logits that the output head's product (gemm_tails.cuh) has left as statistics of pieces of the
// vocabulary: with m_i the largest logit of piece i times log2(e), s_i the sum of 2^(l log2 e - m_i) over it and w_i the same sum weighted
// by its exponents,
//   M = max m_i,  S = sum s_i 2^(m_i - M),  W = sum 2^(m_i - M) (w_i + s_i (m_i - M)),
//   lse = (M + log2 S) ln 2,   log p(target) = l_target - lse,   entropy = (log2 S - W / S) ln 2.
// Compiled without approximate logarithms: the results are fp32 and meant to be.
#include "common.cuh"

namespace ttb {

// Eight rows a block (a sector of neighbouring rows), the pieces dealt out to its 128 groups of eight lanes and joined in a fixed order,
// four at a time under one largest: 1462 pieces are three rounds of loads.
constexpr int JOIN_ROWS = 8, JOIN_GROUPS = 128;

__global__ void __launch_bounds__(JOIN_ROWS * JOIN_GROUPS)
logprobs_join_kernel(const float* __restrict__ part, const float* __restrict__ target_logit, const long long* __restrict__ targets, int slots,
                     long long M, long long V, float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ ent) {
  __shared__ float sm[3][JOIN_GROUPS][JOIN_ROWS];
  const int lane = threadIdx.x % JOIN_ROWS, group = threadIdx.x / JOIN_ROWS;
  const long long row = static_cast<long long>(blockIdx.x) * JOIN_ROWS + lane;
  const long long plane = static_cast<long long>(slots) * M;
  float m = -1e30f, s = 0.f, w = 0.f;
  auto join = [&](float m2, float s2, float w2) {
    const float top = fmaxf(m, m2), a = exp2f(m - top), b = exp2f(m2 - top);
    if (ent) w = a * (w + s * (m - top)) + b * (w2 + s2 * (m2 - top));
    s = s * a + s2 * b;
    m = top;
  };
  if (row < M) {
    constexpr int U = 4;
    for (int i = group; i < slots; i += JOIN_GROUPS * U) {
      float x[U], y[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int slot = i + u * JOIN_GROUPS;
        const float* src = part + slot * M + row;
        x[u] = slot < slots ? src[0] : -1e30f;
        y[u] = slot < slots ? src[plane] : 0.f;
        z[u] = ent && slot < slots ? src[2 * plane] : 0.f;
      }
      float top = x[0], sum = 0.f, dist = 0.f;
#pragma unroll
      for (int u = 1; u < U; ++u) top = fmaxf(top, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float d = x[u] - top, e = exp2f(d);
        sum += e * y[u];
        if (ent) dist += e * (z[u] + y[u] * d);
      }
      join(top, sum, dist);
    }
  }
  sm[0][group][lane] = m; sm[1][group][lane] = s; sm[2][group][lane] = w;
  for (int half = JOIN_GROUPS / 2; half > 0; half /= 2) {
    __syncthreads();
    if (group < half) {
      join(sm[0][group + half][lane], sm[1][group + half][lane], sm[2][group + half][lane]);
      sm[0][group][lane] = m; sm[1][group][lane] = s; sm[2][group][lane] = w;
    }
  }
  if (group != 0 || row >= M) return;
  const float ln2 = 0.6931471805599453f, l2 = log2f(s), all = (m + l2) * ln2;
  const long long t = targets[row];
  logp[row] = t >= 0 && t < V ? target_logit[row] - all : 0.f;
  lse[row] = all;
  if (ent) ent[row] = (l2 - w / s) * ln2;
}

}  // namespace ttb

// part: fp32 [3 with `ent`, else 2][slots][M]
TTB_EXPORT int ttb_logprobs_join(const float* part, const float* target_logit, const long long* targets, int slots, long long M, long long V,
                                 float* logp, float* lse, float* ent, void* stream) {
  using namespace ttb;
  if (M == 0) return 0;
  logprobs_join_kernel<<<static_cast<unsigned>((M + JOIN_ROWS - 1) / JOIN_ROWS), JOIN_ROWS * JOIN_GROUPS, 0, static_cast<cudaStream_t>(stream)>>>(
      part, target_logit, targets, slots, M, V, logp, lse, ent);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
