// A biased linear layer with activation, dropout and residual on a few rows:  C = residual + dropout(act(z)),  z = x W^T + bias.
// One to eight rows leave the tensor cores' tiles of 128 rows empty, and the few tiles that a weight of this size has would each walk the
// whole of K alone; what there is to do is to read the weight once.  So a warp takes CW of its rows (columns of C), its lanes eight
// neighbouring values at a time, multiplied with every row of x in fp32 and added up across the warp in a fixed order.  Bound by the
// latency of its loads where the weight is small, by memory where it is large and rows are one or two, by the products and by reading x again
// above that.  From memory, us (in tiles of the tensor cores' kernel): 1 row 1152 x 1152 3.0 (8.0), 4096 x 4096 8 (16; 5.1 at the rate of a copy),
// 4096 -> 12288 19 (26; 15); 4 rows 3.5 (8.0), 12 (16), 27 (26).
#include "act.cuh"
#include "common.cuh"
#include "philox.cuh"
#include "rowops.cuh"

namespace ttb {

struct RowsParams {
  const __nv_bfloat16 *x, *w, *bias, *residual;
  __nv_bfloat16 *y, *pre;
  long long ldx, ldw, ldr;
  int N, K, act;
  DropoutParams drop;
};

__device__ __forceinline__ uint4 load16_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// KS warps share a column's K, 256 values at a time in turn
template <int M, int CW, int KS>
__global__ void __launch_bounds__(256) linear_rows_kernel(const RowsParams p) {
  __shared__ float part[8][CW * M];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ks = warp % KS;
  const int n0 = (blockIdx.x * (8 / KS) + warp / KS) * CW;
  uint64_t acc[CW][M] = {};                          // sums over even and odd values
  constexpr int U = CW * M >= 16 ? 2 : 4;            // steps whose loads are under way together
  if (n0 < p.N) {
    for (int k0 = ks * 256 + lane * 8; k0 < p.K; k0 += 256 * KS * U) {
      uint4 wv[U][CW];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          const int k = k0 + 256 * KS * u;
          wv[u][c] = make_uint4(0u, 0u, 0u, 0u);
          if (k < p.K && n0 + c < p.N) wv[u][c] = load16_stream(p.w + (n0 + c) * p.ldw + k);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 256 * KS * u;
        if (k >= p.K) break;
        uint64_t f[CW][4];
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          const uint32_t ws[4] = {wv[u][c].x, wv[u][c].y, wv[u][c].z, wv[u][c].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) f[c][j] = f2_pack(__uint_as_float(ws[j] << 16), __uint_as_float(ws[j] & 0xffff0000u));
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const uint4 xu = __ldg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + k));
          const uint32_t xs[4] = {xu.x, xu.y, xu.z, xu.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t x2 = f2_pack(__uint_as_float(xs[j] << 16), __uint_as_float(xs[j] & 0xffff0000u));
#pragma unroll
            for (int c = 0; c < CW; ++c) acc[c][m] = f2_fma(f[c][j], x2, acc[c][m]);
          }
        }
      }
    }
  }
  // lane c M + m goes on with column n0 + c of row m
  float z = 0.f;
#pragma unroll
  for (int c = 0; c < CW; ++c)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float a, b;
      f2_unpack(acc[c][m], a, b);
      const float s = warp_sum(a + b);
      if (lane == c * M + m) z = s;
    }
  if (KS > 1) {
    if (lane < CW * M) part[warp][lane] = z;
    __syncthreads();
    if (ks != 0 || lane >= CW * M) return;
#pragma unroll
    for (int i = 1; i < KS; ++i) z += part[warp + i][lane];
  }
  const int m = lane % M, n = n0 + lane / M;
  if (lane >= CW * M || n >= p.N) return;
  if (p.bias) z += __bfloat162float(p.bias[n]);
  if (p.pre) p.pre[static_cast<long long>(m) * p.N + n] = __float2bfloat16(z);
  float unused = 0.f;
  if (p.act == 1) act_pair<1>(z, unused);
  else if (p.act == 2) act_pair<2>(z, unused);
  if (p.drop.t) {
    const uint4 u = dropout_draws(p.drop.first_row + m, n >> 3, KeysOfSeed(p.drop));
    const uint32_t pair = (n & 4) ? ((n & 2) ? u.w : u.z) : ((n & 2) ? u.y : u.x);
    const uint32_t draw = (n & 1) ? pair >> 16 : pair & 0xffffu;
    z = draw >= p.drop.t ? z * p.drop.scale : 0.f;
  }
  if (p.residual) z += __bfloat162float(p.residual[m * p.ldr + n]);
  p.y[static_cast<long long>(m) * p.N + n] = __float2bfloat16(z);
}

template <int M, int CW>
static void rows_split(const RowsParams& p, int sms, cudaStream_t st) {
  // warps for 16 on every SM: what a warp waits for is its own loads
  const int groups = (p.N + CW - 1) / CW, steps = (p.K + 255) / 256;
  auto go = [&](auto kernel, int ks) { kernel<<<(groups * ks + 7) / 8, 256, 0, st>>>(p); };
  if (groups >= 16 * sms || steps == 1) go(linear_rows_kernel<M, CW, 1>, 1);
  else if (groups >= 8 * sms || steps <= 2) go(linear_rows_kernel<M, CW, 2>, 2);
  else if (groups >= 4 * sms || steps <= 4) go(linear_rows_kernel<M, CW, 4>, 4);
  else go(linear_rows_kernel<M, CW, 8>, 8);
}
template <int M>
static void rows_launch(const RowsParams& p, int sms, cudaStream_t st) {
  // two columns a warp share the loads of x
  if (p.N >= 16 * sms) rows_split<M, 2>(p, sms, st);
  else rows_split<M, 1>(p, sms, st);
}

}  // namespace ttb

// 1 to 8 rows.  x, w, residual: rows of 16-byte aligned bf16; y and pre: [M, N] without gaps; K and N multiples of 8
TTB_EXPORT int ttb_linear_rows(const ttb::GemmArgs* args, void* stream) {
  using namespace ttb;
  const GemmArgs& a = *args;
  if (a.M < 1 || a.M > 8 || (a.K % 8) || (a.N % 8) || (a.lda % 8) || (a.ldb % 8) || a.ldc != a.N || !a.tail || a.tail->drop_t > 65535) return 901;
  if ((reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.B)) & 15) return 902;
  const TailArgs& t = *a.tail;
  const RowsParams p{static_cast<const __nv_bfloat16*>(a.A), static_cast<const __nv_bfloat16*>(a.B), static_cast<const __nv_bfloat16*>(t.bias),
                     static_cast<const __nv_bfloat16*>(a.residual), static_cast<__nv_bfloat16*>(a.C), static_cast<__nv_bfloat16*>(t.pre),
                     a.lda, a.ldb, a.ldr, a.N, a.K, t.act, dropout_params(t.drop_t, t.drop_scale, t.seed, t.seed_dev, t.first_row)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a.M) {
    case 1: rows_launch<1>(p, a.num_sms, st); break;
    case 2: rows_launch<2>(p, a.num_sms, st); break;
    case 3: rows_launch<3>(p, a.num_sms, st); break;
    case 4: rows_launch<4>(p, a.num_sms, st); break;
    case 5: rows_launch<5>(p, a.num_sms, st); break;
    case 6: rows_launch<6>(p, a.num_sms, st); break;
    case 7: rows_launch<7>(p, a.num_sms, st); break;
    default: rows_launch<8>(p, a.num_sms, st); break;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
