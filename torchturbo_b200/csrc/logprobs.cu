// Log-probabilities of rows of logits that the output head's product (gemm_tails.cuh) has left as statistics of pieces of the
// vocabulary: with m_i the largest logit of piece i times log2(e), s_i the sum of 2^(l log2 e - m_i) over it and w_i the same sum weighted
// by its exponents,
//   M = max m_i,  S = sum s_i 2^(m_i - M),  W = sum 2^(m_i - M) (w_i + s_i (m_i - M)),
//   lse = (M + log2 S) ln 2,   log p(target) = l_target - lse,   entropy = (log2 S - W / S) ln 2.
// Compiled without approximate logarithms: the results are fp32 and meant to be.
#include "common.cuh"

namespace ttb {

// Eight rows a block (a sector of neighbouring rows), the pieces dealt out to its 128 groups of eight lanes and joined in a fixed order,
// four at a time under one largest: 1462 pieces are three rounds of loads.  Bound by latency: 61 rows of 1462 pieces 6 us (one warp's lanes
// over 32 rows and a piece at a time: 29), 4096 rows of 1188 27 us of 39 MB, a sixtieth of the product before it.
constexpr int JOIN_ROWS = 8, JOIN_GROUPS = 128;

__global__ void __launch_bounds__(JOIN_ROWS * JOIN_GROUPS)
logprobs_join_kernel(const float* __restrict__ part, const float* __restrict__ target_logit, const long long* __restrict__ targets,
                     const int* __restrict__ rows, const int* __restrict__ count, int row0, int slots, long long M, long long V,
                     float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ ent) {
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
  const bool here = row < M && (!count || row0 + row < *count);
  if (here) {
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
  if (group != 0 || !here) return;
  const float ln2 = 0.6931471805599453f, l2 = log2f(s), all = (m + l2) * ln2;
  const long long t = targets[row];
  logp[rows ? rows[row] : row] = t >= 0 && t < V ? target_logit[row] - all : 0.f;
  lse[row] = all;
  if (ent) ent[row] = (l2 - w / s) * ln2;
}

}  // namespace ttb

namespace ttb {

// Rows that have a target: their places in order, the places' inverse (-1 for the others) and their targets; the others' log-probability is
// zero.  One block: 4096 rows a step, their places by a sum over the threads before; 4096 rows 8.5 us, 8 for copying 3686 of 2048 values.
__global__ void __launch_bounds__(1024)
rows_with_targets_kernel(const long long* __restrict__ targets, long long T, long long V, int* __restrict__ rows, int* __restrict__ place,
                         long long* __restrict__ row_targets, int* __restrict__ count, float* __restrict__ logp) {
  __shared__ int sums[32];
  __shared__ int base;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) base = 0;
  __syncthreads();
  for (long long first = 0; first < T; first += 4096) {
    long long t[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = first + threadIdx.x * 4 + j;
      t[j] = r < T ? targets[r] : -1;
      n += t[j] >= 0 && t[j] < V;
    }
    int before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) sums[warp] = before;
    before -= n;
    __syncthreads();
    int mine = lane < warp ? sums[lane] : 0, all = sums[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    int at = base + mine + before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = first + threadIdx.x * 4 + j;
      if (r >= T) break;
      const bool has = t[j] >= 0 && t[j] < V;
      place[r] = has ? at : -1;
      if (has) {
        rows[at] = static_cast<int>(r);
        row_targets[at++] = t[j];
      } else {
        logp[r] = 0.f;
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// out[j] = x[rows[j]] for j < *count, zeros up to the next multiple of 256 rows (the end of a tile; out has room for it)
__global__ void __launch_bounds__(256)
gather_rows_kernel(const uint4* __restrict__ x, long long ld, const int* __restrict__ rows, const int* __restrict__ count, uint4* __restrict__ out,
                   int vecs) {
  const long long n = *count, end = (n + 255) / 256 * 256;
  for (long long j = blockIdx.x; j < end; j += gridDim.x) {
    const uint4* src = j < n ? x + rows[j] * ld : nullptr;
    for (int c = threadIdx.x; c < vecs; c += 256) out[j * vecs + c] = src ? src[c] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// out[r] = x[place[r]], rounded to bf16, zeros where place[r] < 0
template <typename T>
__global__ void __launch_bounds__(256)
scatter_rows_kernel(const T* __restrict__ x, const int* __restrict__ place, __nv_bfloat16* __restrict__ out, long long R, int cols) {
  for (long long r = blockIdx.x; r < R; r += gridDim.x) {
    const int p = place[r];
    const T* src = x + static_cast<long long>(p < 0 ? 0 : p) * cols;
    for (int c = threadIdx.x * 8; c < cols; c += 256 * 8) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (p >= 0) {
        if (sizeof(T) == 2) {
          u = *reinterpret_cast<const uint4*>(src + c);
        } else {
          const float4 a = *reinterpret_cast<const float4*>(src + c), b = *reinterpret_cast<const float4*>(src + c + 4);
          u = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
        }
      }
      *reinterpret_cast<uint4*>(out + r * cols + c) = u;
    }
  }
}

}  // namespace ttb

// part: fp32 [3 with `ent`, else 2][slots][M].  With `rows`, row j of the product is row rows[j] of `logp`, and those from *count - row0 on are
// not there; lse and ent stay in the product's order.
TTB_EXPORT int ttb_logprobs_join(const float* part, const float* target_logit, const long long* targets, const int* rows, const int* count, int row0,
                                 int slots, long long M, long long V, float* logp, float* lse, float* ent, void* stream) {
  using namespace ttb;
  if (M == 0) return 0;
  logprobs_join_kernel<<<static_cast<unsigned>((M + JOIN_ROWS - 1) / JOIN_ROWS), JOIN_ROWS * JOIN_GROUPS, 0, static_cast<cudaStream_t>(stream)>>>(
      part, target_logit, targets, rows, count, row0, slots, M, V, logp, lse, ent);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// rows, place, row_targets: [T]
TTB_EXPORT int ttb_rows_with_targets(const long long* targets, long long T, long long V, int* rows, int* place, long long* row_targets, int* count,
                                     float* logp, void* stream) {
  using namespace ttb;
  if (T >= (1ll << 31) - 8192) return 901;
  rows_with_targets_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(targets, T, V, rows, place, row_targets, count, logp);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// x: rows of `cols` bf16 values, `ld` apart; out: [T rounded up to 256, cols] without gaps, T at least *count
TTB_EXPORT int ttb_gather_rows(const void* x, long long ld, const int* rows, const int* count, void* out, long long T, int cols, int sms, void* stream) {
  using namespace ttb;
  if (cols % 8 || ld % 8) return 901;
  if (T == 0) return 0;
  const long long blocks = T < 8ll * sms ? T : 8ll * sms;
  gather_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint4*>(x), ld / 8, rows, count,
                                                                                                   static_cast<uint4*>(out), cols / 8);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// x: [.., cols] fp32 or bf16; out: [R, cols] bf16
TTB_EXPORT int ttb_scatter_rows(const void* x, int fp32, const int* place, void* out, long long R, int cols, int sms, void* stream) {
  using namespace ttb;
  if (cols % 8) return 901;
  if (R == 0) return 0;
  const unsigned blocks = static_cast<unsigned>(R < 8ll * sms ? R : 8ll * sms);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp32) scatter_rows_kernel<<<blocks, 256, 0, st>>>(static_cast<const float*>(x), place, static_cast<__nv_bfloat16*>(out), R, cols);
  else scatter_rows_kernel<<<blocks, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), place, static_cast<__nv_bfloat16*>(out), R, cols);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
