// Dropout whose mask is drawn again wherever it is needed (philox.cuh), by itself and in the backward of a biased projection.  What bounds
// them is memory and, nearly as much, the draws: 16384 x 4096 bf16 54 us (a copy 45), with a residual 64 (61.5 at the rate of a copy).
#include <algorithm>

#include "act.cuh"
#include "fastdiv.cuh"
#include "philox.cuh"
#include "rowops.cuh"

namespace ttb {

__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// A block's threads lie over groups of eight columns, and over rows where a row has fewer groups than a block threads; a thread keeps its
// column group and walks rows.  All threads have work where a row is 2048 columns, a part or a multiple of that; 88 % at 1152 and 70 % at
// 4304, 62 % at 2560 and 56 % at 2304.  2^26 bf16 values, TB/s: 1024, 2048, 4096 and 8192 columns 5.3, with a residual 6.5, the backward
// of GELU (erf) 6.1; 1152 columns 4.2, 5.3 and 5.0; 4304 4.0, 5.4 and 5.0; 2560 3.4, 4.7 and 4.3; 2304 3.1, 4.2 and 3.8.
struct Walk {
  int across, per_block, down;      // groups of a row, groups that a block covers, rows that it covers at a time
};
static Walk walk_of(int groups) {
  Walk w{groups, groups < 256 ? groups : 256, 1};
  w.down = 256 / w.per_block;
  return w;
}

// Eight values as they lie in memory
template <typename T>
struct Raw {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) u[i] = load16_here(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
    }
  }
};

// y = residual + dropout(x), rows of whole groups of eight columns; two rows at a time, the next two's loads ahead of their arithmetic.
template <typename T, typename Keys, bool RES>
__global__ void __launch_bounds__(256, sizeof(T) == 2 || !RES ? 3 : 2)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long R, Walk w, const DropoutParams d) {
  const int at = threadIdx.x % w.per_block, g = blockIdx.x * w.per_block + at;
  if (g >= w.across || static_cast<int>(threadIdx.x) >= w.down * w.per_block) return;
  const Keys key(d);
  const uint32_t top = d.t << 16;
  const long long step = static_cast<long long>(gridDim.y) * w.down, stride = static_cast<long long>(w.across) * 8;
  long long row = static_cast<long long>(blockIdx.y) * w.down + threadIdx.x / w.per_block;
  uint32_t high = static_cast<uint32_t>(static_cast<uint64_t>(d.first_row + row) >> 32);
  PhiloxColumn col = philox_column(g, high, key);
  constexpr int U = 2;
  Raw<T> xn[U], rn[U];
  auto load = [&](long long first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (first + u * step >= R) return;
      xn[u].load(x + (first + u * step) * stride + 8 * g);
      if (RES) rn[u].load(residual + (first + u * step) * stride + 8 * g);
    }
  };
  load(row);
  for (; row < R; row += U * step) {
    Raw<T> xs[U], rs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      xs[u] = xn[u];
      if (RES) rs[u] = rn[u];
    }
    load(row + U * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row + u * step >= R) break;
      const uint64_t i = static_cast<uint64_t>(d.first_row + row + u * step);
      if (static_cast<uint32_t>(i >> 32) != high) {
        high = static_cast<uint32_t>(i >> 32);
        col = philox_column(g, high, key);
      }
      float f[8];
      xs[u].values(f);
      dropout8(f, philox(col, philox_row(static_cast<uint32_t>(i), key), key), top, d.scale);
      if (RES) {
        float r[8];
        rs[u].values(r);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] += r[j];
      }
      store8(y + (row + u * step) * stride + 8 * g, f);
    }
  }
}

// The same for rows of any width: eight values in a row of memory belong to two or three groups, so a block draws what its 2048 values
// need once and parks it (C = 1: every value has a group of its own).  Bound by the draws, twenty products each, and the exchange: 4097 x 1003
// fp32 10 us (5 at the rate of a copy), 16000 x 4001 bf16 96 (39; one half of a word read at a time 117).
constexpr int FLAT = 2048;
template <typename T>
__global__ void __launch_bounds__(256)
dropout_flat_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n, int C, FastDiv by_c, int G,
                    FastDiv by_g, const DropoutParams d) {
  extern __shared__ uint4 draws[];
  const KeysOfSeed key(d);
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
  // the values are asked for before the draws, which take as long as they do
  const int k0 = threadIdx.x * 8;
  const long long at = e0 + k0;
  const bool whole = k0 + 8 <= cnt;
  Raw<T> xs, rs;
  if (whole) {
    xs.load(x + at);
    if (residual) rs.load(residual + at);
  }
  int c;
  const int first = c0 >> 3, last = group_of(cnt - 1, c);
  for (int id = first + threadIdx.x; id <= last; id += 256) {
    const int row = by_g(id);
    draws[id - first] = dropout_draws(d.first_row + r0 + row, id - row * G, key);
  }
  __syncthreads();
  if (k0 >= cnt) return;
  int g = group_of(k0, c);
  int row_end = C - c;         // values left in this row
  float f[8], r[8];
  if (whole) {
    xs.values(f);
    if (residual) rs.values(r);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = k0 + j < cnt;
      f[j] = in ? as_float(x[at + j]) : 0.f;
      r[j] = in && residual ? as_float(residual[at + j]) : 0.f;
    }
  }
  const int h0 = (g - first) * 8 + (c & 7);      // place of the first value's draw
  if (row_end >= 8) {
    // of one row: eight halves side by side, from an even one on or an odd one
    const uint32_t* word = reinterpret_cast<const uint32_t*>(draws) + (h0 >> 1);
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = word[j];
    w[4] = (h0 & 1) ? word[4] : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (h0 & 1) ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
    dropout8(f, make_uint4(w[0], w[1], w[2], w[3]), d.t << 16, d.scale);
  } else {
    const uint16_t* half = reinterpret_cast<const uint16_t*>(draws);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = half[(g - first) * 8 + (c & 7)] >= d.t ? f[j] * d.scale : 0.f;
      if (k0 + j + 1 < cnt) {
        ++c;
        if (--row_end == 0) {
          ++g; c = 0; row_end = C;
        } else if ((c & 7) == 0) {
          ++g;
        }
      }
    }
  }
  if (residual) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] += r[j];
  }
  if (whole) {
    store8(y + at, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < cnt) store_scalar(y + at + j, f[j]);
  }
}

// Backward of C = residual + dropout(act(z)):  dz = dropout(dy) act'(z), and its column sums (partial ones per block of rows, reduced by
// colsum_kernel).  `dz` is null where it is dy itself.  Two rows at a time, the next two's loads ahead of their arithmetic; blocks of 256
// threads over 2048 columns, three an SM (blocks as wide as the row, one an SM, had 40 % of the warps and took 159 us for the first
// of these).  8192 x 12288, GELU (erf), dropout and bias 144 us; without dropout 99, without the activation 89 (604, 604 and 403 MB: 92 and
// 62 us at the rate of a copy): the arithmetic of erf and of the draws next to each other is the bound of the first.
template <int ACT, bool DROP, bool SUM, typename Keys>
__global__ void __launch_bounds__(256, 3)
tail_bwd_kernel(const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ z, __nv_bfloat16* __restrict__ dz,
                float* __restrict__ part, int R, Walk w, const DropoutParams d) {
  __shared__ float sums[SUM ? 256 * 8 : 1];
  const int at = threadIdx.x % w.per_block, down = threadIdx.x / w.per_block, g = blockIdx.x * w.per_block + at;
  const bool live = g < w.across && down < w.down;
  float acc[8] = {};
  if (live) {
    const Keys key(d);
    const uint32_t top = d.t << 16;
    const long long stride = static_cast<long long>(w.across) * 8;
    const int step = gridDim.y * w.down;
    int row = blockIdx.y * w.down + down;
    uint32_t high = static_cast<uint32_t>(static_cast<uint64_t>(d.first_row + row) >> 32);
    PhiloxColumn col;
    if (DROP) col = philox_column(g, high, key);
    constexpr int U = 2;
    uint4 du[U], zu[U];
    auto load = [&](int first) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long i = static_cast<long long>(first) + static_cast<long long>(u) * step;
        if (i >= R) return;
        du[u] = load16_here(dy + i * stride + 8 * g);
        if (ACT) zu[u] = load16_here(z + i * stride + 8 * g);
      }
    };
    load(row);
    for (long long at_row = row; at_row < R; at_row += U * step) {
      uint4 ds[U], zs[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ds[u] = du[u];
        if (ACT) zs[u] = zu[u];
      }
      if (at_row + U * step < R) load(static_cast<int>(at_row) + U * step);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long i = at_row + static_cast<long long>(u) * step;
        if (i >= R) break;
        float f[8];
        const uint32_t dw[4] = {ds[u].x, ds[u].y, ds[u].z, ds[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] = __uint_as_float(dw[j] << 16);
          f[2 * j + 1] = __uint_as_float(dw[j] & 0xffff0000u);
        }
        if (DROP) {
          const uint64_t whole = static_cast<uint64_t>(d.first_row + i);
          if (static_cast<uint32_t>(whole >> 32) != high) {
            high = static_cast<uint32_t>(whole >> 32);
            col = philox_column(g, high, key);
          }
          dropout8(f, philox(col, philox_row(static_cast<uint32_t>(whole), key), key), top, d.scale);
        }
        if (ACT) {
          const uint32_t zw[4] = {zs[u].x, zs[u].y, zs[u].z, zs[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float a = __uint_as_float(zw[j] << 16), b = __uint_as_float(zw[j] & 0xffff0000u);
            act_slope_pair<ACT>(a, b);
            f[2 * j] *= a;
            f[2 * j + 1] *= b;
          }
        }
        if (SUM) {
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += f[j];
        }
        if (DROP || ACT) store8(dz + i * stride + 8 * g, f);
      }
    }
  }
  if (!SUM) return;
  // the rows of the block that share a column, in a fixed order
  if (w.down > 1) {
    if (live) store8(sums + (down * w.per_block + at) * 8, acc);
    __syncthreads();
    if (!live || down != 0) return;
    for (int i = 1; i < w.down; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += sums[(i * w.per_block + at) * 8 + j];
    }
  } else if (!live) {
    return;
  }
  store8(part + (static_cast<long long>(blockIdx.y) * w.across + g) * 8, acc);
}

template <typename T>
static void dropout_rows(const void* x, const void* residual, void* y, long long R, int C, const DropoutParams& d, int sms, cudaStream_t st) {
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
  const Walk w = walk_of(C / 8);
  const int bx = (w.across + w.per_block - 1) / w.per_block;
  // three blocks an SM, which is what it holds
  const long long rows = (R + w.down - 1) / w.down;
  const unsigned by = static_cast<unsigned>(std::max<long long>(1, std::min<long long>({rows, 65535, (3ll * sms + bx - 1) / bx})));
  auto go = [&](auto kernel) { kernel<<<dim3(bx, by), 256, 0, st>>>(xs, rs, ys, R, w, d); };
  if (d.seed_dev) rs ? go(dropout_kernel<T, KeysOfSeed, true>) : go(dropout_kernel<T, KeysOfSeed, false>);
  else rs ? go(dropout_kernel<T, KeysOfLaunch, true>) : go(dropout_kernel<T, KeysOfLaunch, false>);
}

}  // namespace ttb

#define STREAM(s) static_cast<cudaStream_t>(s)

// y = residual + dropout(x): [R, C] rows without gaps on 16-byte boundaries, bf16 or fp32; `residual` may be null
TTB_EXPORT int ttb_dropout(const void* x, const void* residual, void* y, int fp32, long long R, int C, unsigned t, float scale,
                           unsigned long long seed, const unsigned long long* seed_dev, long long first_row, int sms, void* stream) {
  using namespace ttb;
  if (R == 0 || C == 0) return 0;
  if (t > 65535) return 903;
  const DropoutParams d = dropout_params(t, scale, seed, seed_dev, first_row);
  if (fp32) dropout_rows<float>(x, residual, y, R, C, d, sms, STREAM(stream));
  else dropout_rows<__nv_bfloat16>(x, residual, y, R, C, d, sms, STREAM(stream));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// Row blocks of ttb_tail_bwd, each of which leaves a row of `part`: three blocks an SM
TTB_EXPORT int ttb_tail_row_blocks(long long R, int C, int sms) {
  using namespace ttb;
  const Walk w = walk_of(C / 8);
  const int bx = (w.across + w.per_block - 1) / w.per_block;
  return static_cast<int>(std::max<long long>(1, std::min<long long>((R + w.down - 1) / w.down, (3ll * sms + bx - 1) / bx)));
}

// part: [row blocks, C] floats, used with `dbias` alone.  dy, z, dz: [R, C] bf16 without gaps on 16-byte boundaries, C % 8 == 0
TTB_EXPORT int ttb_tail_bwd(const void* dy, const void* z, void* dz, float* part, void* dbias, int out_bf16, long long R, int C, int act,
                            unsigned t, float scale, unsigned long long seed, const unsigned long long* seed_dev, long long first_row, int grid,
                            void* stream) {
  using namespace ttb;
  if (C % 8 || act < 0 || act > 2 || (act && !z)) return 901;
  if (t > 65535 || R >= (1ll << 30)) return 903;
  if (R == 0) return 0;
  const DropoutParams d = dropout_params(t, scale, seed, seed_dev, first_row);
  const Walk w = walk_of(C / 8);
  auto go = [&](auto kernel) {
    kernel<<<dim3((w.across + w.per_block - 1) / w.per_block, grid), 256, 0, STREAM(stream)>>>(
        static_cast<const __nv_bfloat16*>(dy), static_cast<const __nv_bfloat16*>(z), static_cast<__nv_bfloat16*>(dz), part, static_cast<int>(R), w, d);
  };
#define TTB_ACT(DROP, SUM, KEYS)                              \
  if (act == 1) go(tail_bwd_kernel<1, DROP, SUM, KEYS>);      \
  else if (act == 2) go(tail_bwd_kernel<2, DROP, SUM, KEYS>); \
  else go(tail_bwd_kernel<0, DROP, SUM, KEYS>);
  if (t && seed_dev) {
    if (dbias) { TTB_ACT(true, true, KeysOfSeed) } else { TTB_ACT(true, false, KeysOfSeed) }
  } else if (t) {
    if (dbias) { TTB_ACT(true, true, KeysOfLaunch) } else { TTB_ACT(true, false, KeysOfLaunch) }
  } else {
    if (dbias) { TTB_ACT(false, true, KeysOfLaunch) } else { TTB_ACT(false, false, KeysOfLaunch) }
  }
#undef TTB_ACT
  if (dbias) colsum(part, dbias, out_bf16, grid, C, STREAM(stream));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
