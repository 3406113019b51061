// Backward of a biased linear layer with a few input features (an adapter's up-projection),  C = residual + dropout(act(z)),  z = x W^T + bias:
//   dz = dropout(dC) act'(z),   dx = dz W,   dW = dz^T x,   db = column sums of dz
// in one walk over dC (and z).  What a row of C holds outweighs what one of x holds a hundred times, so reading dC and z is what it costs:
// dz never leaves the block, as two products that read it again would have it.
//
// A block owns 256 columns and a share of the rows.  Its threads form dz for 32 rows at a time in place of what they copied there, the
// next step's copy under way, and it is an operand of both products: of dx as it lies (every step's sum over the block's columns is
// joined across the warps and goes to memory), of dW transposed (summed over the block's rows in registers).  Sums over blocks of columns,
// and over shares of rows, are added up by linear_narrow_sum_kernel in a fixed order.  The products are 32 x 64 and 256 x 64 wide at most and
// hidden under the loads and draws, so they are mma.sync: an accumulator in TMEM would have to be read back at every step.
// Dropout's factor is left to the sums: without an activation dz is then dC with zeros in it, exact in bf16, and is never unpacked.
//
// 8190 x 16 -> 4096: 18 us and 5 for the sums (67 MB: 10 at the rate of a copy; three passes 37), with dropout 37 and 5 (63), with GELU (erf) too
// 67 together (83).  The first is bound by the latency of a step (wait, barrier, products, joining) at three blocks an SM, the others
// by the instructions of the draws and of the error function, 146 for eight values.  Two blocks an SM with three steps' copies under way 27 and
// 46; dz kept in registers and transposed across the warp (movmatrix) 27 and 47.
#include <algorithm>

#include "act.cuh"
#include "philox.cuh"
#include "rowops.cuh"

namespace ttb {

struct NarrowParams {
  const __nv_bfloat16 *dy, *z, *x, *w;
  long long ldx, ldw;
  float *dx, *dw, *db;         // [column blocks, R, K], [shares, C, K], [shares, C]; null where not wanted
  long long R;
  int C, K, steps;             // steps of 32 rows in a share
  DropoutParams drop;
};
constexpr int NB_COLS = 256, NB_ROWS = 32, NB_LD = NB_COLS + 8;      // rows of the parked dz 528 bytes apart: eight of them lie on distinct banks

template <int KT>
struct NarrowSmem {
  static constexpr int LD = KT + 8;                                  // of x and W, and (in floats) of the sums
  static constexpr int RING = KT <= 32 ? 2 : 3;                      // steps: one at work, the others' loads under way
  static constexpr int TILE = NB_ROWS * NB_LD * 2, X = NB_ROWS * LD * 2, W = NB_COLS * LD * 2, RED = 4 * NB_ROWS * LD * 4;
  static constexpr int TOTAL = RING * (TILE + X) + W + 2 * RED;
  static constexpr int PER_SM = KT <= 16 ? 3 : KT <= 32 ? 2 : 1;     // blocks
};

__device__ __forceinline__ void nb_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void nb_ldm(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void nb_ldm_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// 16 bytes that the copying thread may read after its own wait, others after a barrier as well; zeros in place of what is not there
__device__ __forceinline__ void nb_copy(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void nb_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void nb_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// KT: K rounded up to 16, 32 or 64
template <int KT, int ACT, bool DROP, typename Keys>
__global__ void __launch_bounds__(256, NarrowSmem<KT>::PER_SM) linear_narrow_bwd_kernel(const NarrowParams p) {
  using S = NarrowSmem<KT>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t *tile = smem, *xs = tile + S::RING * S::TILE, *ws = xs + S::RING * S::X;
  float* red = reinterpret_cast<float*>(ws + S::W);
  constexpr int RED = S::RED / 4, NT = KT / 8, AHEAD = S::RING - 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = blockIdx.x * NB_COLS, g = blockIdx.x * (NB_COLS / 8) + lane;      // this thread's eight columns
  const bool live = 8 * g < p.C;
  const long long first = static_cast<long long>(blockIdx.y) * p.steps * NB_ROWS;
  const long long last = first + static_cast<long long>(p.steps) * NB_ROWS < p.R ? first + static_cast<long long>(p.steps) * NB_ROWS : p.R;
  const int xr = tid / NT, xk = tid % NT * 8;      // the eight values of x that this thread brings
  const int mt = warp & 1, quarter = warp >> 1;    // its warp's share of dx: 16 rows, 64 columns

  // copies run AHEAD steps before their use
  const __nv_bfloat16 *from = p.dy + (live ? (first + warp) * p.C + 8 * g : 0), *from_x = p.x + (first + xr) * p.ldx + xk;
  const long long apart = 8ll * p.C, step_x = NB_ROWS * p.ldx;
  int left = static_cast<int>(last - first);      // rows from the next copied step on
  const uint32_t to = smem_u32(tile) + (warp * NB_LD + 8 * lane) * 2, to_x = smem_u32(xs) + (xr * S::LD + xk) * 2;
  auto copy = [&](int b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = live && warp + 8 * i < left;
      nb_copy(to + b * S::TILE + 8 * i * NB_LD * 2, there ? from + i * apart : p.dy, there);
    }
    if (p.dw && tid < NB_ROWS * NT) {
      const bool there = xk < p.K && xr < left;
      nb_copy(to_x + b * S::X, there ? from_x : p.x, there);
    }
    from += 4 * apart;
    from_x += step_x;
    left -= NB_ROWS;
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    copy(j);
    nb_commit();
  }
  // W of these columns, zeros behind its edges, as the operand that a warp's share of dx takes
  for (int i = tid; p.dx && i < NB_COLS * NT; i += 256) {
    const int c = i / NT, k = i % NT * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (c0 + c < p.C && k < p.K) v = *reinterpret_cast<const uint4*>(p.w + static_cast<long long>(c0 + c) * p.ldw + k);
    *reinterpret_cast<uint4*>(ws + (c * S::LD + k) * 2) = v;
  }
  const Keys key(p.drop);
  uint32_t high = 0;
  PhiloxColumn col{};
  if (DROP) {
    high = static_cast<uint32_t>(static_cast<uint64_t>(p.drop.first_row + first) >> 32);
    col = philox_column(g, high, key);
  }
  uint4 zn[ACT ? 4 : 1];
  auto load_z = [&](long long r0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long r = r0 + warp + 8 * i;
      zn[i] = make_uint4(0u, 0u, 0u, 0u);
      if (live && r < last) zn[i] = load16_here(p.z + r * p.C + 8 * g);
    }
  };
  if constexpr (ACT != 0) load_z(first);

  const uint32_t top = p.drop.t << 16;
  // what dropout leaves of two values, but for its factor, which the sums take
  auto kept = [&](uint32_t two, uint32_t draws) { return ((draws << 16) >= top ? two & 0xffffu : 0u) | (draws >= top ? two & 0xffff0000u : 0u); };
  float db[8] = {}, dw[2][NT][4] = {};
  int buf = 0, half = 0;
  bool parked = false;
  // each thread of the sums of one feature, and every 256 / KT-th row
  const int sum_k = tid % KT, sum_r = tid / KT;
  float* sum_to = p.dx + (blockIdx.x * p.R + first + sum_r) * p.K + sum_k;
  const int sum_step = 256 / KT * p.K;
  int sums_left = sum_k < p.K ? static_cast<int>(last - first) - sum_r : 0;
  auto sums_out = [&](int b) {
    const float* src = red + b * RED + sum_r * S::LD + sum_k;
    constexpr int Q = NB_ROWS * S::LD;
#pragma unroll
    for (int i = 0; i < NB_ROWS * KT / 256; ++i, src += 256 / KT * S::LD)
      if (i * (256 / KT) < sums_left) sum_to[i * sum_step] = (src[0] + src[Q]) + (src[2 * Q] + src[3 * Q]);
    sum_to += NB_ROWS * p.K;
    sums_left -= NB_ROWS;
  };
  for (long long r0 = first; r0 < last; r0 += NB_ROWS) {
    const uint32_t at = smem_u32(tile + buf * S::TILE), at_x = smem_u32(xs + buf * S::X);
    nb_wait<AHEAD - 1>();
    // ---- dz of 32 rows, each thread in place of what it copied
    uint4 zu[ACT ? 4 : 1];
    if constexpr (ACT != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) zu[i] = zn[i];
      load_z(r0 + NB_ROWS);
    }
    if (DROP || ACT || p.db) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4* mine = reinterpret_cast<uint4*>(tile + buf * S::TILE + ((warp + 8 * i) * NB_LD + 8 * lane) * 2);
        uint4 du = *mine;
        if (DROP) {
          const uint64_t whole = static_cast<uint64_t>(p.drop.first_row + r0 + warp + 8 * i);
          if (static_cast<uint32_t>(whole >> 32) != high) {
            high = static_cast<uint32_t>(whole >> 32);
            col = philox_column(g, high, key);
          }
          const uint4 u = philox(col, philox_row(static_cast<uint32_t>(whole), key), key);
          du = make_uint4(kept(du.x, u.x), kept(du.y, u.y), kept(du.z, u.z), kept(du.w, u.w));
        }
        if (ACT || p.db) {
          float f[8];
          const uint32_t dv[4] = {du.x, du.y, du.z, du.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f[2 * j] = __uint_as_float(dv[j] << 16);
            f[2 * j + 1] = __uint_as_float(dv[j] & 0xffff0000u);
          }
          if (ACT) {
            const uint32_t zv[4] = {zu[i].x, zu[i].y, zu[i].z, zu[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float a = __uint_as_float(zv[j] << 16), b = __uint_as_float(zv[j] & 0xffff0000u);
              act_slope_pair<ACT>(a, b);
              f[2 * j] *= a;
              f[2 * j + 1] *= b;
            }
            du = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) db[j] += f[j];
        }
        if (DROP || ACT) *mine = du;
      }
    }
    // One barrier a step: behind it everyone has done with the step before, whose place takes the copies of the step AHEAD of this one, and
    // its parked sums are there
    __syncthreads();
    copy(buf == 0 ? AHEAD : buf - 1);
    nb_commit();
    if (parked && p.dx) sums_out(half ^ 1);
    parked = true;
    // ---- dx: 16 rows x K over 64 columns a warp
    if (p.dx) {
      float acc[NT][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t a[4];
        nb_ldm(a, at + ((16 * mt + (lane & 15)) * NB_LD + 64 * quarter + 16 * ks + (lane >> 4) * 8) * 2);
#pragma unroll
        for (int nt = 0; nt < NT; nt += 2) {
          uint32_t b[4];
          nb_ldm_t(b, smem_u32(ws) + ((64 * quarter + 16 * ks + (lane & 15)) * S::LD + 8 * nt + (lane >> 4) * 8) * 2);
          nb_mma(acc[nt], a, b[0], b[1]);
          nb_mma(acc[nt + 1], a, b[2], b[3]);
        }
      }
      float* out = red + half * RED + (quarter * NB_ROWS + 16 * mt + (lane >> 2)) * S::LD + 2 * (lane & 3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        *reinterpret_cast<float2*>(out + 8 * nt) = make_float2(acc[nt][0], acc[nt][1]);
        *reinterpret_cast<float2*>(out + 8 * S::LD + 8 * nt) = make_float2(acc[nt][2], acc[nt][3]);
      }
    }
    // ---- dW: 32 columns x K over 32 rows a warp
    if (p.dw) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t a[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
          nb_ldm_t(a[m], at + ((16 * ks + (lane & 7) + (lane >> 4) * 8) * NB_LD + 32 * warp + 16 * m + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
        for (int nt = 0; nt < NT; nt += 2) {
          uint32_t b[4];
          nb_ldm_t(b, at_x + ((16 * ks + (lane & 15)) * S::LD + 8 * nt + (lane >> 4) * 8) * 2);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            nb_mma(dw[m][nt], a[m], b[0], b[1]);
            nb_mma(dw[m][nt + 1], a[m], b[2], b[3]);
          }
        }
      }
    }
    buf = buf == AHEAD ? 0 : buf + 1;
    half ^= 1;
  }
  nb_wait<0>();
  __syncthreads();
  if (parked && p.dx) sums_out(half ^ 1);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 32 * warp + 16 * m + (lane >> 2) + 8 * h, k = 8 * nt + 2 * (lane & 3);
        if (p.dw && c < p.C && k < p.K)
          *reinterpret_cast<float2*>(p.dw + (static_cast<long long>(blockIdx.y) * p.C + c) * p.K + k) = make_float2(dw[m][nt][2 * h], dw[m][nt][2 * h + 1]);
      }
  if (!p.db) return;
  // the eight warps' sums of a column, in order
  __syncthreads();
  float* part = red;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[warp * NB_COLS + 8 * lane + j] = db[j];
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += part[i * NB_COLS + tid];
  if (c0 + tid < p.C) p.db[static_cast<long long>(blockIdx.y) * p.C + c0 + tid] = s;
}

struct NarrowSums {
  const float *dx, *dw, *db;
  __nv_bfloat16 *out_x, *out_w;
  void* out_b;
  int b_bf16, blocks, shares;
  float scale;
  long long nx, nw, nb;      // pairs of values
};
__global__ void __launch_bounds__(256) linear_narrow_sum_kernel(const NarrowSums p) {
  long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const float* src;
  long long n;
  int parts, which;
  if (i < p.nx) {
    src = p.dx; n = p.nx; parts = p.blocks; which = 0;
  } else if ((i -= p.nx) < p.nw) {
    src = p.dw; n = p.nw; parts = p.shares; which = 1;
  } else if ((i -= p.nw) < p.nb) {
    src = p.db; n = p.nb; parts = p.shares; which = 2;
  } else {
    return;
  }
  float2 s = make_float2(0.f, 0.f);
  const float2* at = reinterpret_cast<const float2*>(src) + i;
  for (int j = 0; j < parts; j += 16, at += 16 * n) {      // sixteen loads under way
    float2 v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = j + u < parts ? __ldg(at + u * n) : make_float2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      s.x += v[u].x;
      s.y += v[u].y;
    }
  }
  s.x *= p.scale;
  s.y *= p.scale;
  const uint32_t u = pack_bf16(s.x, s.y);
  if (which == 0) reinterpret_cast<uint32_t*>(p.out_x)[i] = u;
  else if (which == 1) reinterpret_cast<uint32_t*>(p.out_w)[i] = u;
  else if (p.b_bf16) reinterpret_cast<uint32_t*>(p.out_b)[i] = u;
  else reinterpret_cast<float2*>(p.out_b)[i] = s;
}

// Blocks of columns, shares of rows (as many as the SMs hold) and steps of 32 rows in a share
struct NarrowPlan {
  int blocks, shares, steps;
};
static NarrowPlan narrow_plan(long long R, int C, int K, int sms) {
  NarrowPlan q;
  q.blocks = (C + NB_COLS - 1) / NB_COLS;
  const int per_sm = K <= 16 ? NarrowSmem<16>::PER_SM : K <= 32 ? NarrowSmem<32>::PER_SM : NarrowSmem<64>::PER_SM;
  const long long steps = (R + NB_ROWS - 1) / NB_ROWS, most = std::max<long long>(1, static_cast<long long>(per_sm) * sms / q.blocks);
  q.steps = static_cast<int>((steps + std::min(most, steps) - 1) / std::min(most, steps));
  q.shares = static_cast<int>((steps + q.steps - 1) / q.steps);
  return q;
}

template <int KT, int ACT, bool DROP, typename Keys>
static int narrow_launch(const NarrowParams& p, const NarrowPlan& q, cudaStream_t st) {
  auto kernel = linear_narrow_bwd_kernel<KT, ACT, DROP, Keys>;
  constexpr int smem = NarrowSmem<KT>::TOTAL;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return 300 + static_cast<int>(e);
  kernel<<<dim3(q.blocks, q.shares), 256, smem, st>>>(p);
  return 0;
}
template <int KT, int ACT>
static int narrow_drop(const NarrowParams& p, const NarrowPlan& q, cudaStream_t st) {
  if (!p.drop.t) return narrow_launch<KT, ACT, false, KeysOfLaunch>(p, q, st);
  if (p.drop.seed_dev) return narrow_launch<KT, ACT, true, KeysOfSeed>(p, q, st);
  return narrow_launch<KT, ACT, true, KeysOfLaunch>(p, q, st);
}
template <int KT>
static int narrow_act(const NarrowParams& p, const NarrowPlan& q, int act, cudaStream_t st) {
  if (act == 1) return narrow_drop<KT, 1>(p, q, st);
  if (act == 2) return narrow_drop<KT, 2>(p, q, st);
  return narrow_drop<KT, 0>(p, q, st);
}

// ---------------------------------------------------------------------------------------------
// The layer itself with up to 16 input features, where C is small or an activation is applied: one walk over its rows.  A warp owns 32 columns, whose weights stay in
// registers, and multiplies 16 rows at a time, the next 16 rows' loads under way.  The columns are dealt to the products' columns so that
// a thread ends up with eight neighbouring ones of a row: 16 bytes of the residual and of C, and what one draw of the dropout is for.
// Bound by its loads and stores; no TMEM to fill and to read, no tile to wait for.  us, and by the tiles of gemm.cu: 200 x 16 -> 1152 2.1 (5.0), with dropout
// and residual 2.5 (5.9); 16384 x 16 -> 1024 11 (17), 19 (28), with GELU (tanh) and pre-activations 14 (30).
// ---------------------------------------------------------------------------------------------
struct NarrowFwd {
  const __nv_bfloat16 *x, *w, *bias, *residual;
  __nv_bfloat16 *y, *pre;
  long long ldx, ldw, ldr, R;
  int N, K, across, per_block, down;      // warps across a row, of a block, and rows of warps in it
  DropoutParams drop;
};

template <int ACT, bool DROP, typename Keys>
__global__ void __launch_bounds__(256, 3) linear_narrow_fwd_kernel(const NarrowFwd p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int place = blockIdx.x * p.per_block + warp % p.per_block;
  if (warp >= p.per_block * p.down || place >= p.across) return;
  const int col = 32 * place + 8 * t;
  const bool live = col < p.N;
  // column 2 t + e of the j-th product is column 8 t + 2 j + e of the warp's
  uint32_t wf[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = 32 * place + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) wf[j][h] = c < p.N && 8 * h < p.K ? __ldg(reinterpret_cast<const uint32_t*>(p.w + c * p.ldw + 8 * h + 2 * t)) : 0u;
  }
  uint4 bias = make_uint4(0u, 0u, 0u, 0u);
  if (p.bias && live) bias = __ldg(reinterpret_cast<const uint4*>(p.bias + col));
  const Keys key(p.drop);
  const int step = gridDim.y * p.down * 16, first = (blockIdx.y * p.down + warp / p.per_block) * 16 + g;      // this thread's first row
  uint64_t row = static_cast<uint64_t>(p.drop.first_row) + first;      // its place for the dropout
  uint32_t high = static_cast<uint32_t>(row >> 32);
  PhiloxColumn column{};
  if (DROP) column = philox_column(col >> 3, high, key);
  // addresses move on by steps: products of 64 bits for every row took as many instructions as all the rest
  long long left = p.R - first;                  // rows from this thread's on
  const __nv_bfloat16 *x = p.x + first * p.ldx + 2 * t, *residual = p.residual + first * p.ldr + col;
  const long long out0 = static_cast<long long>(first) * p.N + col;
  __nv_bfloat16 *y = p.y + out0, *pre = p.pre + out0;
  const long long x_8 = 8 * p.ldx, x_step = step * p.ldx, r_8 = 8 * p.ldr, r_step = step * p.ldr, y_8 = 8ll * p.N, y_step = static_cast<long long>(step) * p.N;
  const bool second = p.K > 8;
  uint4 rn[2];
  uint32_t xn[4];
  auto load = [&](long long there) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = 8 * i < there;
      if (p.residual && live && in) rn[i] = load16_here(residual + i * r_8);
      xn[i] = in ? __ldg(reinterpret_cast<const uint32_t*>(x + i * x_8)) : 0u;
      xn[i + 2] = in && second ? __ldg(reinterpret_cast<const uint32_t*>(x + i * x_8 + 8)) : 0u;
    }
    x += x_step;
    residual += r_step;
  };
  load(left);
  // whole warps go on for as long as one of their rows is there
  for (; left + g > 0; left -= step, y += y_step, pre += y_step, row += step) {
    uint4 rs[2];
    float acc[4][4] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) rs[i] = rn[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) nb_mma(acc[j], xn, wf[j][0], wf[j][1]);
    load(left - step);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!live || 8 * i >= left) continue;
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = acc[j][2 * i];
        f[2 * j + 1] = acc[j][2 * i + 1];
      }
      auto add = [&](const uint4& v) {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] += __uint_as_float(u[j] << 16);
          f[2 * j + 1] += __uint_as_float(u[j] & 0xffff0000u);
        }
      };
      if (p.bias) add(bias);
      if (p.pre) store8(pre + i * y_8, f);
      if (ACT) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) act_pair<ACT>(f[j], f[j + 1]);
      }
      if (DROP) {
        const uint64_t whole = row + 8 * i;
        if (static_cast<uint32_t>(whole >> 32) != high) {
          high = static_cast<uint32_t>(whole >> 32);
          column = philox_column(col >> 3, high, key);
        }
        dropout8(f, philox(column, philox_row(static_cast<uint32_t>(whole), key), key), p.drop.t << 16, p.drop.scale);
      }
      if (p.residual) add(rs[i]);
      store8(y + i * y_8, f);
    }
  }
}

template <int ACT>
static void narrow_fwd(const NarrowFwd& p, int sms, cudaStream_t st) {
  const int bx = (p.across + p.per_block - 1) / p.per_block;
  const long long rows = (p.R + 16 * p.down - 1) / (16 * p.down);
  const unsigned by = static_cast<unsigned>(std::max<long long>(1, std::min<long long>({rows, 65535, (3ll * sms + bx - 1) / bx})));
  auto go = [&](auto kernel) { kernel<<<dim3(bx, by), 256, 0, st>>>(p); };
  if (!p.drop.t) go(linear_narrow_fwd_kernel<ACT, false, KeysOfLaunch>);
  else if (p.drop.seed_dev) go(linear_narrow_fwd_kernel<ACT, true, KeysOfSeed>);
  else go(linear_narrow_fwd_kernel<ACT, true, KeysOfLaunch>);
}

}  // namespace ttb

// x, w, residual: rows of bf16 values on 16-byte boundaries; y and pre: [M, N] without gaps; N % 8 == 0, K 8 or 16
TTB_EXPORT int ttb_linear_narrow(const ttb::GemmArgs* args, void* stream) {
  using namespace ttb;
  const GemmArgs& a = *args;
  if (a.M < 1 || a.N < 1 || (a.K != 8 && a.K != 16) || (a.N % 8) || (a.lda % 8) || (a.ldb % 8) || (a.ldr % 8) || a.ldc != a.N || !a.tail ||
      a.tail->act < 0 || a.tail->act > 2 || a.tail->drop_t > 65535)
    return 901;
  const TailArgs& t = *a.tail;
  if ((reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C) | reinterpret_cast<uintptr_t>(t.bias) |
       reinterpret_cast<uintptr_t>(t.pre) | reinterpret_cast<uintptr_t>(a.residual)) & 15)
    return 902;
  const int across = (a.N + 31) / 32, per_block = across < 8 ? across : 8;
  const NarrowFwd p{static_cast<const __nv_bfloat16*>(a.A), static_cast<const __nv_bfloat16*>(a.B), static_cast<const __nv_bfloat16*>(t.bias),
                    static_cast<const __nv_bfloat16*>(a.residual), static_cast<__nv_bfloat16*>(a.C), static_cast<__nv_bfloat16*>(t.pre),
                    a.lda, a.ldb, a.ldr, a.M, a.N, a.K, across, per_block, 8 / per_block,
                    dropout_params(t.drop_t, t.drop_scale, t.seed, t.seed_dev, t.first_row)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (t.act == 1) narrow_fwd<1>(p, a.num_sms, st);
  else if (t.act == 2) narrow_fwd<2>(p, a.num_sms, st);
  else narrow_fwd<0>(p, a.num_sms, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

// fp32 values that ttb_linear_narrow_bwd keeps its partial sums in
TTB_EXPORT int ttb_linear_narrow_parts(long long R, int C, int K, int sms, long long* parts) {
  const ttb::NarrowPlan q = ttb::narrow_plan(R, C, K, sms);
  *parts = q.blocks * R * K + static_cast<long long>(q.shares) * C * (K + 1);
  return 0;
}

// dy, z: [R, C] bf16 without gaps; x: [R, K] and w: [C, K], rows ldx and ldw apart; all on 16-byte boundaries; C % 8 == 0, K % 8 == 0, K <= 64.
// dx [R, K] and dw [C, K] bf16, db [C] bf16 or fp32; each null unless wanted
TTB_EXPORT int ttb_linear_narrow_bwd(const void* dy, const void* z, const void* x, long long ldx, const void* w, long long ldw, void* dx, void* dw, void* db,
                                     int db_bf16, float* parts, long long R, int C, int K, int act, unsigned t, float scale, unsigned long long seed,
                                     const unsigned long long* seed_dev, long long first_row, int sms, void* stream) {
  using namespace ttb;
  if (C <= 0 || K <= 0 || C % 8 || K % 8 || K > 64 || ldx % 8 || ldw % 8 || act < 0 || act > 2 || (act && !z)) return 901;
  if (t > 65535 || R <= 0 || R >= (1ll << 30)) return 903;
  const NarrowPlan q = narrow_plan(R, C, K, sms);
  if (q.shares > 65535) return 903;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  float *px = parts, *pw = px + q.blocks * R * K, *pb = pw + static_cast<long long>(q.shares) * C * K;
  const NarrowParams p{static_cast<const __nv_bfloat16*>(dy), static_cast<const __nv_bfloat16*>(z), static_cast<const __nv_bfloat16*>(x),
                       static_cast<const __nv_bfloat16*>(w), ldx, ldw, dx ? px : nullptr, dw ? pw : nullptr, db ? pb : nullptr, R, C, K, q.steps,
                       dropout_params(t, scale, seed, seed_dev, first_row)};
  const int r = K <= 16 ? narrow_act<16>(p, q, act, st) : K <= 32 ? narrow_act<32>(p, q, act, st) : narrow_act<64>(p, q, act, st);
  if (r) return r;
  const NarrowSums s{px, pw, pb, static_cast<__nv_bfloat16*>(dx), static_cast<__nv_bfloat16*>(dw), db, db_bf16, q.blocks, q.shares, t ? scale : 1.f,
                     dx ? R * K / 2 : 0, dw ? static_cast<long long>(C) * K / 2 : 0, db ? C / 2 : 0};
  linear_narrow_sum_kernel<<<static_cast<unsigned>((s.nx + s.nw + s.nb + 255) / 256), 256, 0, st>>>(s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
