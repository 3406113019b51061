// Epilogues of gemm.cu for what follows a biased projection and for rows of logits that are not stored.  Included by gemm.cu alone.
//
//   tail_store    C = residual + dropout(act(z)), z = product + bias; z itself is kept in bf16 where the backward needs it (it reads z for
//                 act'(z) only).  Everything up to C's one rounding stays fp32.  Under long sums the tail is hidden; of short ones it is the
//                 whole kernel, bound by the latency of its arithmetic: sixteen warps instead of eight took a sum of 16 products, 8190 x 4096 of them,
//                 with dropout and residual from 52 to 48 us (residual and all at the rate of a copy: 31).  3001 x 1152 -> 4304 with bias, GELU (tanh) and
//                 pre-activations 30 us in short runs, with GELU (erf) 32, with the bias alone 26.
//   tail_stats    of each row's logits in this tile and half of its columns: largest, sum of exponentials, and for the entropy their sum
//                 weighted by the distance from the largest (logprobs.cu joins them).  All in powers of two: with m the largest times
//                 log2(e) as rounded to fp32, d = l log2(e) - m is one fma, 2^d one instruction, and log2 sum 2^(l log2 e) = m + log2 s is
//                 exact in m whatever its rounding was.  Nearly hidden under sums of 512: 4096 x 2048 x 151936 under the power cap 1877 us,
//                 1358 TFLOP/s, where the product that stores its results takes 1925.
//   tail_dlogits  gradient of the logits, formed again from the same operands:  p = 2^(l log2 e - lse log2 e),
//                 dl = g (1[target] - p) - e p (l - lse + H), rounded to bf16, the type in which the two products behind it take it.  Of few
//                 rows one value, the target's, is most of a row, and its rounding would not average out: what it left out goes to a
//                 second plane, as further rows of those products.  A piece of 4096 x 2048 x 50688 568 us, the plain product of the same size 561.
#pragma once

namespace ttb {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void add8(float (&f)[8], const uint4& u) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  f[0] += a.x; f[1] += a.y; f[2] += b.x; f[3] += b.y; f[4] += c.x; f[5] += c.y; f[6] += d.x; f[7] += d.y;
}
__device__ __forceinline__ void add_bias8(float (&f)[8], const __nv_bfloat16* bias, int col) {
  if (bias) add8(f, __ldg(reinterpret_cast<const uint4*>(bias + col)));
}
// What an epilogue thread reads of its row (one row a thread) before the accumulator is there
template <int EPI>
struct TailRow {
  __device__ __forceinline__ void fetch(const GemmParams&, int, int) {}
};
template <>
struct TailRow<EPI_TAIL> {
  uint4 res[2], bias[2];      // of 16 columns
  const __nv_bfloat16* src;
  long long row;
  __device__ __forceinline__ void fetch_bias(const GemmParams& p, int col) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (p.tail.bias && col + 8 * i < p.N) bias[i] = load16_here(p.tail.bias + col + 8 * i);
  }
  __device__ __forceinline__ void fetch_residual(const GemmParams& p, int col) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (src && col + 8 * i < p.N) res[i] = load16_here(src + col + 8 * i);
  }
  // `cols` columns of a row of the next tile into the L2: an epilogue of short sums is over before they would come from memory
  __device__ __forceinline__ void ahead(const GemmParams& p, int r, int col, int cols) {
    if (!p.residual || r >= p.M) return;
    for (int c = col; c < col + cols && c < p.N; c += 64)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.residual + static_cast<long long>(r) * p.ldr + c));
  }
  __device__ __forceinline__ void fetch(const GemmParams& p, int r, int col, int cols) {
    row = r;
    src = p.residual && r < p.M ? p.residual + static_cast<long long>(r) * p.ldr : nullptr;
#pragma unroll
    for (int i = 0; i < 2; ++i) res[i] = bias[i] = make_uint4(0u, 0u, 0u, 0u);
    if (cols > 0) {
      fetch_residual(p, col);
      fetch_bias(p, col);
    }
  }
};
template <>
struct TailRow<EPI_LSE> {
  long long target;
  __device__ __forceinline__ void fetch(const GemmParams& p, int r, int rows) { target = r < rows ? __ldg(p.tail.targets + r) : -1; }
};
template <>
struct TailRow<EPI_DLOGITS> {
  long long target;      // column of this product, or one that it does not have
  float lse2, g, e, shift;
  __device__ __forceinline__ void fetch(const GemmParams& p, int r, int rows) {
    const TailParams& q = p.tail;
    target = -1;
    lse2 = g = e = shift = 0.f;
    if (r >= rows) return;
    const int from = q.rows ? __ldg(q.rows + r) : r;      // row of the caller's gradients
    const long long t = __ldg(q.targets + r);
    if (t >= 0 && t < q.vocab) {
      target = t - q.first_col;
      g = q.dlogp ? __ldg(q.dlogp + from) : 0.f;
    }
    const float lse = __ldg(q.lse + r);
    lse2 = lse * LOG2E;
    if (q.dent) {
      e = __ldg(q.dent + from);
      shift = __ldg(q.ent + r);
    }
  }
};

// 16 values plus 16 packed ones
__device__ __forceinline__ void add16(float (&f)[16], const uint4 (&u)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float& a = f[8 * i + 2 * j];
      float& b = f[8 * i + 2 * j + 1];
      f2_unpack(f2_add(f2_pack(a, b), f2_pack(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u))), a, b);
    }
  }
}
template <int ACT>
__device__ __forceinline__ void act16(float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) act_pair<ACT>(f[i], f[i + 1]);
}

// `at`: TMEM address of this warp's rows and first column, `first` that column in C, `cols` how many it has (64 or none).  Sixteen columns
// at a time; pre-activations are parked and stored first, the result from the same accumulator after them.
template <typename Release>
__device__ __forceinline__ void tail_store(const GemmParams& p, const CUtensorMap& tmC, const CUtensorMap& tmZ, TailRow<EPI_TAIL>& tr, uint8_t* stage_at,
                                           uint32_t at, int first, int cols, int row_base, int lane, Release release) {
  const TailParams& q = p.tail;
  if (cols <= 0 || first >= p.N || row_base >= p.M) {      // uniform across the warp
    release();
    return;
  }
  const KeysOfSeed key(q.drop);
  const uint64_t place = static_cast<uint64_t>(q.drop.first_row + tr.row);
  PhiloxRow mine{};
  if (q.drop.t) mine = philox_row(static_cast<uint32_t>(place), key);
  const uint32_t st = smem_u32(stage_at);
#pragma unroll 1
  for (int pass = q.has_pre ? 0 : 1; pass < 2; ++pass) {
    // the copy engine has read what was parked before
    if (lane == 0) bulk_wait_read_all();
    __syncwarp();
#pragma unroll 1
    for (int c = 0; c < 64; c += 16) {
      const int col0 = first + c;
      float f[16];
      {
        uint32_t v[16];
        tmem_ld_32x32b_x16(at + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
      }
      if (pass == 1 && c == 48) release();
      if (q.bias) add16(f, tr.bias);
      if (pass == 1) {
        if (q.act == 1) act16<1>(f);
        else if (q.act == 2) act16<2>(f);
        if (q.drop.t) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            dropout8(f + 8 * i, philox(philox_column((col0 >> 3) + i, static_cast<uint32_t>(place >> 32), key), mine, key), q.drop.t << 16, q.drop.scale);
        }
        if (p.residual) add16(f, tr.res);
      }
      if (c < 48 || pass == 0) tr.fetch_bias(p, c < 48 ? col0 + 16 : first);
      if (c < 48 && pass == 1) tr.fetch_residual(p, col0 + 16);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        st_shared_v4(epi_piece_addr(st, lane, (c >> 3) + i), pack_bf16(f[8 * i], f[8 * i + 1]), pack_bf16(f[8 * i + 2], f[8 * i + 3]),
                     pack_bf16(f[8 * i + 4], f[8 * i + 5]), pack_bf16(f[8 * i + 6], f[8 * i + 7]));
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(pass ? &tmC : &tmZ, stage_at, first, row_base, 0);
      bulk_commit_group();
    }
  }
}

// The tensor cores' fp32 sums are cut off, not rounded, at every addition: after 2048 products of random signs they are 1.4e-6 of their
// size too near to zero, all of them to the same side, and the bias grows with the length (1024: 6.6e-7, 512: 3.1e-7).
// Log-probabilities leave in fp32, so their sums are run over LSE_RUN k-blocks at a time and the runs are added up in registers, rounded.
// 4096 x 2048 x 151936 under the power cap: one run 1815 us, runs of 16 blocks 1816, of 8 blocks 1877.  Eight, for 3 % of the time: runs of 16
// are twice as far off as fp32 sums of rounded products (6.8e-7 and 1.9e-7 of log-probabilities in the 2-norm).
constexpr int LSE_RUN = 8;

template <int BN>
__device__ __forceinline__ void tail_add(float (&sum)[BN / 2], uint32_t at, int cols) {
#pragma unroll
  for (int c = 0; c < BN / 2; c += 16) {
    if (c >= cols) break;
    uint32_t v[16];
    tmem_ld_32x32b_x16(at + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 2)
      f2_unpack(f2_add(f2_pack(sum[c + i], sum[c + i + 1]), f2_pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1]))), sum[c + i], sum[c + i + 1]);
  }
}

template <int BN>
__device__ __forceinline__ void tail_stats(const GemmParams& p, const TailRow<EPI_LSE>& tr, float (&l)[BN / 2], int first, int cols, int slot,
                                           int row) {
  const TailParams& q = p.tail;
  if (cols < BN / 2) {
#pragma unroll
    for (int i = 0; i < BN / 2; ++i)
      if (i >= cols) l[i] = -1e30f;
  }
  const long long hit = tr.target - first;
  if (hit >= 0 && hit < cols) {
    float at = 0.f;
#pragma unroll
    for (int i = 0; i < BN / 2; ++i)
      if (hit == i) at = l[i];
    q.target_logit[row] = at;
  }
  float big = fmaxf(l[0], l[1]);
#pragma unroll
  for (int i = 2; i < BN / 2; i += 2) big = fmax3(big, l[i], l[i + 1]);
  const float m = fmaxf(big * LOG2E, -1e30f);   // of no columns, or where all are -infinity: a sum of zero
  float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
  const uint64_t log2e = f2_pack(LOG2E, LOG2E), down = f2_pack(-m, -m);
  auto pass = [&](bool entropy) {
#pragma unroll
    for (int i = 0; i < BN / 2; i += 2) {
      float d0, d1;
      f2_unpack(f2_fma(f2_pack(l[i], l[i + 1]), log2e, down), d0, d1);
      const float e0 = exp2_approx(d0), e1 = exp2_approx(d1);
      s0 += e0; s1 += e1;
      if (entropy) { w0 = fmaf(e0, d0, w0); w1 = fmaf(e1, d1, w1); }
    }
  };
  if (q.entropy) pass(true);
  else pass(false);
  if (row < p.M) {
    const long long slots = 2ll * p.n_tiles, plane = slots * p.M;
    float* dst = q.part + slot * static_cast<long long>(p.M) + row;
    dst[0] = m;
    dst[plane] = s0 + s1;
    if (q.entropy) dst[2 * plane] = w0 + w1;
  }
}

template <int BN, typename Release>
__device__ __forceinline__ void tail_dlogits(const GemmParams& p, const CUtensorMap& tmC, const TailRow<EPI_DLOGITS>& tr, uint8_t* stage_at,
                                             uint32_t at, int first, int row_base, int lane, Release release) {
  const uint32_t sy = smem_u32(stage_at);
  const bool silent = tr.g == 0.f && tr.e == 0.f;     // zeros, whatever the row holds
  const float ln2 = 0.6931471805599453f;
  bool held = true;
#pragma unroll 1
  for (int c = 0; c < BN / 2; c += 64) {
    const int col0 = first + c;
    if (col0 >= p.N || row_base >= p.M) break;      // uniform across the warp
    uint32_t v[2][32];
    tmem_ld_32x32b_x32(at + c, v[0]);
    tmem_ld_32x32b_x32(at + c + 32, v[1]);
    tmem_ld_wait();
    if (c + 64 >= BN / 2) {
      release();
      held = false;
    }
    const int hit = tr.target >= col0 && tr.target < col0 + 64 ? static_cast<int>(tr.target - col0) : -1;
    // (the rounded value, and with `rest` what its rounding left out)
    auto park = [&](bool rest) {
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
      if (silent) {
#pragma unroll
        for (int i = 0; i < 8; ++i) st_shared_v4(epi_piece_addr(sy, lane, i), 0u, 0u, 0u, 0u);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float d = fmaf(__uint_as_float(v[i >> 2][(8 * i + j) & 31]), LOG2E, -tr.lse2);
            const float pr = exp2_approx(d);
            f[j] = -pr * (p.tail.dent ? fmaf(tr.e, fmaf(d, ln2, tr.shift), tr.g) : tr.g);
            if (hit == 8 * i + j) f[j] += tr.g;
          }
          if (rest) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] -= __bfloat162float(__float2bfloat16(f[j]));
          }
          const uint4 y = pack8(f);
          st_shared_v4(epi_piece_addr(sy, lane, i), y.x, y.y, y.z, y.w);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(&tmC, stage_at, col0, row_base, rest ? 1 : 0);
        bulk_commit_group();
      }
    };
    park(false);
    if (p.tail.has_pre) park(true);
  }
  if (held) release();
}

}  // namespace ttb
