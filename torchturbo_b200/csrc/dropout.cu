// Dropout whose mask is drawn again wherever it is needed (philox.cuh), by itself and in the backward of a biased projection.
#include <algorithm>

#include "act.cuh"
#include "fastdiv.cuh"
#include "philox.cuh"
#include "rowops.cuh"

namespace ttb {

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// y = residual + dropout(x), rows of whole groups of eight columns, a group a thread.
template <typename T>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, int groups, FastDiv by_row, int per_row, DropoutParams d) {
  const PhiloxKey key = dropout_key(d);
  for (int i = blockIdx.x * 256 + threadIdx.x; i < groups; i += gridDim.x * 256) {
    const int row = by_row(i), g = i - row * per_row;
    float f[8];
    load8(x + 8ll * i, f);
    dropout8(f, dropout_draws(d.first_row + row, g, key), d.t, d.scale);
    if (residual) {
      float r[8];
      load8(residual + 8ll * i, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += r[j];
    }
    store8(y + 8ll * i, f);
  }
}

// The same for rows of any width: eight values in a row of memory belong to two or three groups, so a block draws what its 2048 values
// need once and parks it (C = 1: every value has a group of its own).
constexpr int FLAT = 2048;
template <typename T>
__global__ void __launch_bounds__(256)
dropout_flat_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n, int C, FastDiv by_c, int G,
                    FastDiv by_g, DropoutParams d) {
  extern __shared__ uint4 draws[];
  const PhiloxKey key = dropout_key(d);
  const long long e0 = static_cast<long long>(blockIdx.x) * FLAT;
  const int cnt = static_cast<int>(n - e0 < FLAT ? n - e0 : FLAT);
  const long long r0 = e0 / C;
  const int c0 = static_cast<int>(e0 - r0 * C);
  // group of the block's k-th value, counted from the first group of its first row
  auto group_of = [&](int k, int& c) {
    const int row = by_c(c0 + k);
    c = c0 + k - row * C;
    return row * G + (c >> 3);
  };
  int c;
  const int first = c0 >> 3, last = group_of(cnt - 1, c);
  for (int id = first + threadIdx.x; id <= last; id += 256) {
    const int row = by_g(id);
    draws[id - first] = dropout_draws(d.first_row + r0 + row, id - row * G, key);
  }
  __syncthreads();
  const uint16_t* half = reinterpret_cast<const uint16_t*>(draws);
  const int k0 = threadIdx.x * 8;
  if (k0 >= cnt) return;
  const long long at = e0 + k0;
  int g = group_of(k0, c);
  int row_end = C - c;         // values left in this row
  float f[8], r[8];
  const bool whole = k0 + 8 <= cnt;
  if (whole) {
    load8(x + at, f);
    if (residual) load8(residual + at, r);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = k0 + j < cnt;
      f[j] = in ? as_float(x[at + j]) : 0.f;
      r[j] = in && residual ? as_float(residual[at + j]) : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = half[(g - first) * 8 + (c & 7)];
    f[j] = u >= d.t ? f[j] * d.scale : 0.f;
    if (residual) f[j] += r[j];
    if (k0 + j + 1 < cnt) {
      ++c;
      if (--row_end == 0) {
        ++g; c = 0; row_end = C;
      } else if ((c & 7) == 0) {
        ++g;
      }
    }
  }
  if (whole) {
    store8(y + at, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < cnt) store_scalar(y + at + j, f[j]);
  }
}

// Backward of C = residual + dropout(act(z)):  dz = dropout(dy) act'(z), and its column sums.  Blocks walk rows of up to 8192 columns
// (blockIdx.y: which), eight columns a thread, the next row's loads ahead of this one's arithmetic, as the backward of the separate
// bias and activation does; `dz` is null where it is dy itself, `part` where no sums are wanted.
template <int ACT, bool DROP>
__global__ void __launch_bounds__(1024)
tail_bwd_kernel(const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ z, __nv_bfloat16* __restrict__ dz,
                float* __restrict__ part, long long R, int C, DropoutParams d) {
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (c >= C) return;
  PhiloxKey key{0u, 0u};
  if (DROP) key = dropout_key(d);
  float acc[8] = {};
  uint4 du = make_uint4(0, 0, 0, 0), zu = du;
  auto load = [&](long long row) {
    if (row >= R) return;
    du = *reinterpret_cast<const uint4*>(dy + row * C + c);
    if (ACT) zu = *reinterpret_cast<const uint4*>(z + row * C + c);
  };
  load(blockIdx.x);
  for (long long row = blockIdx.x; row < R; row += gridDim.x) {
    const uint32_t ds[4] = {du.x, du.y, du.z, du.w}, zs[4] = {zu.x, zu.y, zu.z, zu.w};
    load(row + gridDim.x);
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 g = unpack_bf16(ds[j]);
      f[2 * j] = g.x; f[2 * j + 1] = g.y;
    }
    if (DROP) dropout8(f, dropout_draws(d.first_row + row, c >> 3, key), d.t, d.scale);
    if (ACT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack_bf16(zs[j]);
        f[2 * j] *= act_slope<ACT>(v.x);
        f[2 * j + 1] *= act_slope<ACT>(v.y);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += f[j];
    if (dz) store8(dz + row * C + c, f);
  }
  if (!part) return;
  store8(part + static_cast<long long>(blockIdx.x) * C + c, acc);
}

template <typename T>
static void dropout_rows(const void* x, const void* residual, void* y, long long R, int C, DropoutParams d, int sms, cudaStream_t st) {
  const T *xs = static_cast<const T*>(x), *rs = static_cast<const T*>(residual);
  T* ys = static_cast<T*>(y);
  if (C % 8) {
    const int G = (C + 7) / 8;
    const long long n = R * C;
    // groups of 2048 values: one for every eight and one more for each row that they touch
    const int slots = FLAT / 8 + FLAT / C + 4;
    dropout_flat_kernel<T><<<static_cast<unsigned>((n + FLAT - 1) / FLAT), 256, slots * sizeof(uint4), st>>>(xs, rs, ys, n, C, fast_div(C), G,
                                                                                                             fast_div(G), d);
    return;
  }
  const int per_row = C / 8;
  const long long most = std::max<long long>(1, ((1ll << 31) - (1 << 24)) / per_row);
  for (long long a = 0; a < R; a += most, d.first_row += most) {
    const int groups = static_cast<int>(std::min(most, R - a) * per_row);
    const int blocks = std::min((groups + 255) / 256, sms * 8);
    dropout_kernel<T><<<blocks, 256, 0, st>>>(xs + a * C, rs ? rs + a * C : nullptr, ys + a * C, groups, fast_div(per_row), per_row, d);
  }
}

}  // namespace ttb

#define STREAM(s) static_cast<cudaStream_t>(s)

// y = residual + dropout(x): [R, C] rows without gaps on 16-byte boundaries, bf16 or fp32; `residual` may be null
TTB_EXPORT int ttb_dropout(const void* x, const void* residual, void* y, int fp32, long long R, int C, unsigned t, float scale,
                           unsigned long long seed, const unsigned long long* seed_dev, long long first_row, int sms, void* stream) {
  using namespace ttb;
  if (R == 0 || C == 0) return 0;
  const DropoutParams d{t, scale, seed, seed_dev, first_row};
  if (fp32) dropout_rows<float>(x, residual, y, R, C, d, sms, STREAM(stream));
  else dropout_rows<__nv_bfloat16>(x, residual, y, R, C, d, sms, STREAM(stream));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// part: grid * C floats, with `dbias` null it is not used.  dy, z, dz: [R, C] bf16 without gaps on 16-byte boundaries, C % 8 == 0, C <= 16384
TTB_EXPORT int ttb_tail_bwd(const void* dy, const void* z, void* dz, float* part, void* dbias, int out_bf16, long long R, int C, int act,
                            unsigned t, float scale, unsigned long long seed, const unsigned long long* seed_dev, long long first_row, int grid,
                            void* stream) {
  using namespace ttb;
  if (C % 8 || act < 0 || act > 2 || (act && !z)) return 901;
  if (C > 16384) return 902;
  if (R == 0) return 0;
  if (grid > R) grid = static_cast<int>(R);
  const DropoutParams d{t, scale, seed, seed_dev, first_row};
  const int width = C > 8192 ? (C + 15) / 16 * 8 : C, threads = (width / 8 + 31) / 32 * 32;
  auto go = [&](auto kernel) {
    kernel<<<dim3(grid, C > 8192 ? 2 : 1), threads, 0, STREAM(stream)>>>(
        static_cast<const __nv_bfloat16*>(dy), static_cast<const __nv_bfloat16*>(z), static_cast<__nv_bfloat16*>(dz), dbias ? part : nullptr, R, C, d);
  };
  if (t) {
    if (act == 1) go(tail_bwd_kernel<1, true>);
    else if (act == 2) go(tail_bwd_kernel<2, true>);
    else go(tail_bwd_kernel<0, true>);
  } else {
    if (act == 1) go(tail_bwd_kernel<1, false>);
    else if (act == 2) go(tail_bwd_kernel<2, false>);
    else go(tail_bwd_kernel<0, false>);
  }
  if (dbias) colsum(part, dbias, out_bf16, grid, C, STREAM(stream));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
