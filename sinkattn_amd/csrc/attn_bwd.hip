// Backward pass of the block-sparse attention for gfx950, with recomputed probabilities.
//
// With S = scale Q K^T on the listed 128x128 tiles, the saved row log-sum-exp lse and the gradient
// dO of the output (and dlse of the lse):
//     P = exp(S - lse)       dP = dO V^T       delta = rowsum(dO * O) - dlse
//     dS = P * (dP - delta)  dQ = scale dS K   dK = scale dS^T Q   dV = P^T dO
// The compensation keys (kd, vd) are further columns of S with ln(gap) added.
//
// Two kernels of one shape.  A wave owns columns, 16 or 32 rows of one side held in registers, and
// streams the rows of the other side through LDS:
//     dQ    columns = queries (Q, dO), streamed = the listed keys (K, V):
//           S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T
//     dK/dV columns = keys (K, V), streamed = the queries that list them (Q, dO):
//           S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// The accumulators of the first two products hold a column per lane and the streamed rows in the
// registers, which is the B operand of the others, so P and dS never leave the registers.  S and dP
// are computed by both kernels (seven products in place of five): every gradient is then summed
// by one group in a fixed order, without atomics, and results do not change from run to run.  (Five products in all would
// need dS kept between them.  By arithmetic, not tried: 16-bit dS is 64 KB of traffic a tile, 13 ns of the chip's memory
// against 7 ns for two products; in fp32 it is 128 KB, 26 ns against 54, so there it could pay.)
// What bounds it, bf16, D = 128, 12 heads of 32760 tokens with 20% of the tiles: the power limit.  dQ takes 1.44 ms
// (1.33 PFLOP/s of its three products), dK/dV 2.04 ms (1.26 of its four) on a card whose library product of 8192^3 reaches
// 1.19 PFLOP/s, 1.56 and 2.17 ms on one with 1.13, there at 1.72-1.76 GHz of 2.4 with the matrix cores busy 63-66% of the
// cycles.  f16 takes 1.65 + 2.32 ms on the first (library 1.18).  Short lists (24 heads of 8190 tokens with pooled keys: 0.31 + 0.39
// ms, 1.18 PFLOP/s) pay some 17 us per round of work-groups for the columns' operands and results.
// The dQ kernel runs first and leaves each row's lse (in log2 units) and -delta in the workspace.

#include "common.h"
#include "kernels.h"

namespace sa {

// One side's rows in memory: base pointer of a (b, h) and row stride in elements.
struct Rows {
  const char* base;
  int64_t stride;
};

template <int ES>
__device__ __forceinline__ Rows head_rows(const void* p, const int64_t (&s)[4], int b, int h) {
  return Rows{(const char*)p + ((int64_t)b * s[0] + (int64_t)h * s[1]) * ES, s[2]};
}

// ------------------------------------------------------------------------------------
// bf16/f16.  A group of four waves takes a block of 128 columns, 32 (two 16-column tiles ct) per
// wave, and streams 64 rows per step: both operands' rows come by buffer DMA into one of two pairs of
// LDS tiles while the other pair is multiplied.  All products run on v_mfma_f32_16x16x32:
//     s[rt][ct], u[rt][ct]   A = 16 rows rt of Y1 / Y2, B = the columns' X1 / X2 in registers
//     acc[n][dt][ct]         A = Y^T by transpose reads, B = dS / P of 32 rows from s and u
// Lane l holds column 16 ct + l % 16 in all of them and rows 4 (l / 16) + i, i < 4, of a row tile.
// The tiles are read both ways, so the chunk swizzle of BwdGeom serves row and transpose reads.
// P and dS are rounded to the operands' type for the second pair of products (half a step each, as the
// forward does with P).  In f16, values near one would leave most of the range unused and
// probabilities of long rows (and with them dS) would fall below its normal numbers, so both are
// multiplied by powers of two, which the stores divide out: P by 2^kPShift, and dS by a factor per
// column that is lowered whenever a step's largest |dS| would pass kDsLimit (an exact rescaling of
// the accumulator, as of a softmax's running maximum).
// 32 columns a wave, because one wave per SIMD with 64 (half the LDS reads per product) had its accumulators in the
// other half of the register file, with a move around every product: 2.8 ms for dK/dV above, 2.1 as it is.  D = 64 runs
// three waves per SIMD and is bound by VALU work, an exponential and some six other instructions per 256 flops (2 x 16
// heads of 8100 tokens, 25%, fp16: 0.21 + 0.29 ms, 0.93 PFLOP/s; bf16 0.19 + 0.24; D = 32 0.15 + 0.19 and 0.13 + 0.15).
// ------------------------------------------------------------------------------------
constexpr float kPShift = 14.f;        // log2; P is at most 1, or barely above by the lse's rounding
constexpr float kDsStart = 30.f;       // log2 of a column's first dS factor
constexpr float kDsLimit = 32768.f;    // of a scaled dS
constexpr float kDsTarget = 11.f;      // log2 of the largest scaled dS after a lowering

template <int D>
struct BwdGeom {
  static constexpr int kRow = 2 * D;              // bytes of a tile row
  static constexpr int kChunks = D / 8;           // 16-byte chunks of a row
  static constexpr int kCopyRows = 64 / kChunks;  // rows of one wave's copy instruction
  // Chunk swizzle: the 8 lanes of a row read that LDS serves at a time (rows 0-7 or 8-15, one chunk) touch
  // 128 distinct bytes modulo 128, the 32 of a transpose read (32 bytes of 8 rows) 256 modulo 256: no bank
  // conflicts (a swizzle of distinct bytes modulo 256 for 16 rows cost the row reads 40% more LDS cycles).
  // Adding 16 to a row changes nothing.
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (D == 128) return ((row & 3) << 1) | ((row >> 2) & 1) | ((((row >> 2) ^ (row >> 3)) & 1) << 3);
    if constexpr (D == 64) return row & 7;
    return (row >> 1) & 3;
  }
};

// 4 bytes per lane from rsrc + voffset into LDS at lds_wave_base + 4 lane.
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, SA_LDS void* lds_wave_base, uint32_t voffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_wave_base, 4, voffset, 0, 0, 0);
}

// Where a row's lse and -delta are in the workspace: blocks of four rows, lse then -delta, so that 32
// rows are one 4-byte copy of a wave and a lane's four rows two 16-byte reads.
__device__ __forceinline__ int64_t row_slot(int64_t row) { return (row >> 2) * 8 + (row & 3); }

// Per-lane offsets in a tile (bytes) of the reads.  Those of k-step ks or d-tile dt differ from the first
// one's in the chunk bits alone: an exclusive or, also with 32 rows added.
template <int D>
struct BwdLanes {
  uint32_t row0;  // row read: row l % 16, chunk 4 ks + l / 16
  uint32_t tr0;   // transpose read: rows 4 (l / 16) + (l % 16) / 4, columns 16 dt + 4 (l % 4)
};

template <int D>
__device__ __forceinline__ BwdLanes<D> bwd_lanes(int lane) {
  using G = BwdGeom<D>;
  const int g = lane >> 4, sl = lane & 15, trow = 4 * g + (sl >> 2);
  return BwdLanes<D>{(uint32_t)(sl * G::kRow + ((g ^ G::swz(sl)) * 16)),
                     (uint32_t)(trow * G::kRow + ((((sl & 3) >> 1) ^ G::swz(trow)) * 16) + (sl & 1) * 8)};
}

// The A operand of 32 streamed rows from the transpose-read address `p` of the first of them.
template <int D>
__device__ __forceinline__ u32x4 tr_read(SA_LDS char* p) {
  const u32x2 y0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SA_LDS v4i16*)p));
  const u32x2 y1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SA_LDS v4i16*)(p + 16 * 2 * D)));
  return u32x4{y0[0], y0[1], y1[0], y1[1]};
}

// 32 columns' results, scaled by f, through this wave's 64 D bytes of LDS so that whole rows are stored.
template <int CT, int D>
__device__ __forceinline__ void store_columns(char* base, int64_t stride, int own0, int Nown, const f32x4 (&acc)[D / 16][2],
                                              const float (&f)[2], SA_LDS char* buf, int lane) {
  using G = BwdGeom<D>;
  const int g = lane >> 4, sl = lane & 15;
#pragma unroll
  for (int ct = 0; ct < 2; ++ct)
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      u32x2 w;
      w[0] = pack2<CT>(acc[dt][ct][0] * f[ct], acc[dt][ct][1] * f[ct]);
      w[1] = pack2<CT>(acc[dt][ct][2] * f[ct], acc[dt][ct][3] * f[ct]);
      const int chunk = (2 * dt + (g >> 1)) ^ G::swz(sl);
      *(SA_LDS u32x2*)(buf + (16 * ct + sl) * G::kRow + chunk * 16 + (g & 1) * 8) = w;
    }
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0) only
#pragma unroll
  for (int i = 0; i < 32 / G::kCopyRows; ++i) {
    const int row = G::kCopyRows * i + lane / G::kChunks, ch = lane % G::kChunks;
    const u32x4 val = *(SA_LDS const u32x4*)(buf + row * G::kRow + ((ch ^ G::swz(row)) * 16));
    if (own0 + row < Nown) *reinterpret_cast<u32x4*>(base + (int64_t)(own0 + row) * stride * 2 + ch * 16) = val;
  }
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // the reads are back: buf is free again
}

// The same in fp32, 64 bytes of a row at a time from the registers.
template <int D>
__device__ __forceinline__ void store_columns_f32(char* base, int64_t stride, int own0, int Nown, const f32x4 (&acc)[D / 16][2],
                                                  const float (&f)[2], int lane) {
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    const int own = own0 + 16 * ct + (lane & 15);
    if (own >= Nown) continue;
    float* to = (float*)base + (int64_t)own * stride + 4 * (lane >> 4);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(to + 16 * dt) = acc[dt][ct] * f[ct];
  }
}

template <int CT>
__device__ __forceinline__ float unpack16(uint32_t w, int hi) {
  const uint32_t x = hi ? w >> 16 : w & 0xffffu;
  return CT == kBF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x);
}

// Rows of a step, and whether the columns' X2 stays in LDS instead of registers.  dK and dV at D = 128
// take 128 registers and K 32 more: V in registers would leave too few for two waves per SIMD.
template <int D, bool KEYS>
struct BwdShape {
  static constexpr bool kX2Lds = KEYS && D == 128;
  static constexpr int kStep = kX2Lds ? 32 : 64;
  static constexpr int kTile = kStep * BwdGeom<D>::kRow;
};

// 32 streamed rows, `at` bytes into tile y1 (Y2's a tile behind; their lse and -delta at `rows` where the
// columns are keys), against the wave's 32 columns.  S starts at `start`.
template <int CT, int D, bool KEYS>
__device__ __forceinline__ void bwd_rows32(SA_LDS char* y1, uint32_t at, SA_LDS const char* rows, SA_LDS const char* x2,
                                           const BwdLanes<D>& L, const u32x4 (&b1)[2][D / 32], const u32x4 (&b2)[2][D / 32],
                                           f32x4 (&acc)[KEYS ? 2 : 1][D / 16][2], const float (&lse2)[2],
                                           const float (&ndelta)[2], float (&m)[2], float bias, float c2,
                                           const f32x4 (&start)[2], int g) {
  using G = BwdGeom<D>;
  using S = BwdShape<D, KEYS>;
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int NR = (KEYS ? 2 : 1) * DT;     // transpose reads: dV's products first, then dK's / dQ's
  constexpr int AHEAD = 4, TAHEAD = NR < 2 ? NR : 2;  // reads issued ahead of their products
  f32x4 s[2][2], u[2][2];
  u32x4 p[2], ds[2];
  // dP starts at -delta, as the first products' addend
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    f32x4 rd = f32x4{};
    if constexpr (KEYS) rd = *(SA_LDS const f32x4*)(rows + (4 * rt + g) * 32 + 16);
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      s[rt][ct] = KEYS ? f32x4{} : start[rt];
      u[rt][ct] = KEYS ? rd : f32x4{ndelta[ct], ndelta[ct], ndelta[ct], ndelta[ct]};
    }
  }
  {
    // reads: per k-step both row tiles of Y1; then per k-step (X2's two column tiles and) both of Y2
    constexpr int PER = S::kX2Lds ? 4 : 2, N1 = 2 * KS, N = N1 + PER * KS;
    u32x4 r[N];
    auto read = [&](int i) {
      const bool second = i >= N1;
      const int ks = second ? (i - N1) / PER : i / 2, j = second ? (i - N1) % PER - (PER - 2) : i % 2;
      const uint32_t flip = (uint32_t)(ks * 64);
      if (j < 0) return *(SA_LDS const u32x4*)(x2 + (L.row0 ^ flip) + (j + 2) * 16 * G::kRow);
      return *(SA_LDS const u32x4*)(y1 + ((at + L.row0) ^ flip) + (second ? S::kTile : 0) + j * 16 * G::kRow);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) r[i] = read(i);
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD + (KEYS ? 2 : 0), 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool second = i >= N1;
      const int ks = second ? (i - N1) / PER : i / 2, j = second ? (i - N1) % PER - (PER - 2) : i % 2;
      if (i + AHEAD < N) {
        r[i + AHEAD] = read(i + AHEAD);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      if (j < 0) continue;
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        if (!second) s[j][ct] = mfma16x16x32<CT>(r[i], b1[ct][ks], s[j][ct]);
        else u[j][ct] = mfma16x16x32<CT>(r[i], S::kX2Lds ? r[N1 + PER * ks + ct] : b2[ct][ks], u[j][ct]);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  u32x4 r[NR];
  auto tread = [&](int i) { return tr_read<D>(y1 + ((at + L.tr0) ^ (uint32_t)(i % DT * 32)) + (NR - i > DT ? S::kTile : 0)); };
#pragma unroll
  for (int i = 0; i < TAHEAD; ++i) r[i] = tread(i);
  // s becomes P, u dS
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    f32x4 rl;  // KEYS: the rows' lse
    if constexpr (KEYS) rl = *(SA_LDS const f32x4*)(rows + (4 * rt + g) * 32);
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      float shift = bias;
      if constexpr (CT == kF16) shift += KEYS ? kPShift : m[ct];
      const float fds = CT == kF16 && KEYS ? fast_exp2(m[ct] - kPShift) : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[rt][ct][i] = fast_exp2(__builtin_fmaf(s[rt][ct][i], c2, shift - (KEYS ? rl[i] : lse2[ct])));
        u[rt][ct][i] *= s[rt][ct][i];
        if constexpr (CT == kF16 && KEYS) u[rt][ct][i] *= fds;
      }
    }
  }
  if constexpr (CT == kF16) {
    float mx[2];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      const f32x4 x = u[0][ct], y = u[1][ct];
      mx[ct] = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                     fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
    }
    if (__builtin_amdgcn_ballot_w64(fmaxf(mx[0], mx[1]) > kDsLimit) != 0) {
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        const float top = max_col16(mx[ct]);
        if (top > kDsLimit && top < pos_inf()) {  // (not for an infinite or NaN gradient)
          const float down = kDsTarget - ceilf(__log2f(top)), f = fast_exp2(down);
          m[ct] += down;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[0][dt][ct] *= f;
          u[0][ct] *= f;
          u[1][ct] *= f;
        }
      }
    }
  }
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (KEYS) p[ct][2 * rt + e] = pack2<CT>(s[rt][ct][2 * e], s[rt][ct][2 * e + 1]);
        ds[ct][2 * rt + e] = pack2<CT>(u[rt][ct][2 * e], u[rt][ct][2 * e + 1]);
      }
  if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);  // 1.5% faster at D = 128, nothing at 64
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int n = NR - i > DT ? 1 : 0;
    if (i + TAHEAD < NR) r[i + TAHEAD] = tread(i + TAHEAD);
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) acc[n][i % DT][ct] = mfma16x16x32<CT>(r[i], n ? p[ct] : ds[ct], acc[n][i % DT][ct]);
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    if (i + TAHEAD < NR) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
}

// Rows past the last query, zero as they come, become copies of it.  Their lse of +inf makes P 0 from every score but
// NaN, which a zero row would have with an infinite key.  `at` is the byte of a row's chunk in the tile.
template <int STEP, int CHUNKS, class At>
__device__ __forceinline__ void repeat_last_row(SA_LDS char* tile, int left, int tid, At at) {
  if (left >= STEP) return;
#pragma unroll 1
  for (int i = tid; i < (STEP - left) * CHUNKS; i += 256)
    *(SA_LDS u32x4*)(tile + at(left + i / CHUNKS, i % CHUNKS)) = *(SA_LDS const u32x4*)(tile + at(left - 1, i % CHUNKS));
  drain_then_barrier();
}

// First of the `blocks` blocks of part p.
__device__ __forceinline__ int part_begin(int blocks, int p, int parts) { return (int)((int64_t)blocks * p / parts); }

// A query block's parts: of q_share blocks at least, q_parts of them at most.
__device__ __forceinline__ int q_item_parts(const BwdArgs& a, int item) {
  int blocks = ((const SA_CONST int32_t*)a.counts)[item];
  if (a.comp_qblocks > 0 && item % a.nqb < a.comp_qblocks) blocks += (a.Nd + 127) >> 7;
  return max(1, min(a.q_parts, (blocks + a.q_share - 1) / a.q_share));
}

// Cuts the long lists of the key blocks (one work-group).  A block whose list is longer than an even share of all lists for the
// groups that run at a time gets as many parts as shares: with the parts first in the launch, no group outlasts
// the others by more than about a share.  (Lists as long as that are the rule for sink keys, which every query block
// lists, and for the pooled keys.)  There are at most twice as many parts as shares, which k_slots allows for.
// Where whole lists all run at once, a larger share may be the better one: a part costs its sums' way through memory
// (of all parts together, about 60 ns each), a tile more on the longest list about kTileParts as much, and parts that do
// not all run at once a second round.  Whole calls with this choice of share against the even share, D = 128: [1,40,1101]
// 88 against 104 us, [1,12,4000] 141 and 161, [2,12,2500] 143 and 162, [1,30,1101] with pooled keys 84 and 89, equal
// at [1,12,2048] and [1,1,16000], and 54 against 53 at [1,8,2000,64].  kTileParts = 96 against 24 and 384: [1,24,1000] 62, 65 and
// 66; [1,40,1101] 88, 96 and 88; [1,30,1101] with pooled keys 84, 92 and 84; [1,1,16000] 105, 117 and 105; [1,4,8190] with pooled keys
// 154, 165 and 154; [1,12,5000] with them 214, 204 and 215; [1,16,2500,32] 60, 60 and 64.
constexpr int kTileParts = 96;

__device__ void plan_key_parts(const BwdArgs& a) {
  __shared__ int64_t sums[4];
  __shared__ int scan[4], ncut[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nsparse = a.B * a.H * a.nkb, n = nsparse + a.B * a.H * ((a.Nd + 127) >> 7);
  for (int i = tid; i < a.k_slots; i += 256) a.slot_item[i] = a.extra_slot[i] = -1;
  int64_t sum = 0;
  for (int i = tid; i < n; i += 256) sum += i < nsparse ? a.kcounts[i] : a.comp_qblocks;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += ((int64_t)__shfl_xor((int)(sum >> 32), o, 64) << 32) + (uint32_t)__shfl_xor((int)sum, o, 64);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  const int64_t total = sums[0] + sums[1] + sums[2] + sums[3];
  int share = max(1, (int)((total + a.k_shares - 1) / a.k_shares));
  if (a.k_one_round && n <= a.k_shares) {
    int best = 1 << 30;
    for (int s = share; s * kTileParts < best; s += max(1, s / 8)) {
      int groups = 0, cut = 0;  // of this share
      for (int i = tid; i < n; i += 256) {
        const int parts = max(1, ((i < nsparse ? a.kcounts[i] : a.comp_qblocks) + s - 1) / s);
        groups += parts;
        cut += parts > 1 ? parts : 0;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        groups += __shfl_xor(groups, o, 64);
        cut += __shfl_xor(cut, o, 64);
      }
      if (lane == 0) {
        scan[wave] = groups;
        ncut[wave] = cut;
      }
      __syncthreads();
      groups = scan[0] + scan[1] + scan[2] + scan[3];
      cut = ncut[0] + ncut[1] + ncut[2] + ncut[3];
      __syncthreads();
      const int cost = s * kTileParts * (groups > a.k_shares ? 2 : 1) + cut;
      if (cost < best) {
        best = cost;
        share = s;
      }
    }
  }
  int base = 0, cuts = 0;  // slots and lists so far
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + tid;
    const int cnt = i >= n ? 0 : i < nsparse ? a.kcounts[i] : a.comp_qblocks;
    const int parts = cnt > share ? (cnt + share - 1) / share : 0;
    int incl = parts;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const uint64_t cut = __ballot(parts > 0);
    if (lane == 63) {
      scan[wave] = incl;
      ncut[wave] = __popcll(cut);
    }
    __syncthreads();
    int at = base + incl - parts, before = cuts + __popcll(cut & ((1ull << lane) - 1ull));
    for (int w = 0; w < wave; ++w) {
      at += scan[w];
      before += ncut[w];
    }
    if (i < n) a.split_base[i] = parts > 0 ? at : -1;
    for (int p = 0; p < parts; ++p) {
      a.slot_item[at + p] = i;
      a.slot_part[at + p] = p | parts << 16;
      if (p == 0) a.cut_slot[1 + before] = at;
      // the parts but the first, packed, so that they go to the XCDs in turn
      if (p > 0) a.extra_slot[at + p - before - 1] = at + p;
    }
    base += scan[0] + scan[1] + scan[2] + scan[3];
    cuts += ncut[0] + ncut[1] + ncut[2] + ncut[3];
    __syncthreads();
  }
  if (tid == 0) {
    a.cut_slot[0] = cuts;
    a.cut_slot[1 + a.k_slots] = (base - cuts + kXcds - 1) / kXcds * kXcds;
  }
}

// What a work-group takes: a block of columns and a share of its list.  item < 0: nothing.
struct BwdItem {
  int item, part, parts, slot0;  // slot0: the item's first partial sum
  bool of_pooled;                // a block of the pooled keys
};

// Queries: q_parts groups per order slot, on the slot's XCD (work-group i runs on XCD i % 8), after eight groups of
// which the first finds the key blocks to cut.  Keys: first the parts (but the first) of those, then the pooled keys'
// blocks, as many per XCD, in order, so that an XCD's L2 holds one head's Q and dO at a time, then the
// order's `slots` slots.
template <bool KEYS>
__device__ __forceinline__ BwdItem bwd_item(const BwdArgs& a, int blk, int slots) {
  BwdItem w{-1, 0, 1, 0, false};
  if constexpr (KEYS) {
    const int nsparse = a.B * a.H * a.nkb;
    const int pooled_items = a.B * a.H * ((a.Nd + 127) >> 7), pooled_per = (pooled_items + kXcds - 1) / kXcds;
    // (blocks without work at the launch's end)
    const int extras = a.k_slots > 0 ? __builtin_amdgcn_readfirstlane(a.cut_slot[1 + a.k_slots]) : 0;
    if (blk < extras) {
      const int slot = __builtin_amdgcn_readfirstlane(a.extra_slot[blk]);
      if (slot < 0) return w;
      const int pp = __builtin_amdgcn_readfirstlane(a.slot_part[slot]);
      w.item = __builtin_amdgcn_readfirstlane(a.slot_item[slot]);
      w.part = pp & 0xffff;
      w.parts = pp >> 16;
      w.slot0 = slot - w.part;
    } else {
      blk -= extras;
      if (blk < pooled_per * kXcds) {
        const int i = blk % kXcds * pooled_per + blk / kXcds;
        if (i >= pooled_items) return w;
        w.item = nsparse + i;
      } else {
        blk -= pooled_per * kXcds;
        if (blk >= slots) return w;
        w.item = __builtin_amdgcn_readfirstlane(a.korder ? a.korder[blk] : blk);
        if (w.item < 0) return w;
      }
      const int sb = a.k_slots > 0 ? __builtin_amdgcn_readfirstlane(a.split_base[w.item]) : -1;
      if (sb >= 0) {
        w.slot0 = sb;
        w.parts = __builtin_amdgcn_readfirstlane(a.slot_part[sb]) >> 16;
      }
    }
    w.of_pooled = w.item >= nsparse;
    if (w.of_pooled) w.item -= nsparse;
  } else {
    if (blk < kXcds) {
      if (blk == 0 && a.k_slots > 0) plan_key_parts(a);
      return w;
    }
    blk -= kXcds;
    // A slot's parts follow each other.  Where all run at once, the first parts of all slots come first: of parts in turn, those
    // without work would leave their neighbours two to a CU and other CUs idle (19 -> 24 us for 270 lists of one tile; whole calls
    // in turn instead: [1,30,1101] with pooled keys 84 -> 92 us, [1,24,700] with them 60 -> 66, [1,16,2500,32] 60 -> 64, but
    // [1,12,4000] 141 -> 138 and [1,1,16000] 105 -> 103).
    const int rounded = (slots + kXcds - 1) / kXcds * kXcds;
    const bool first_ones = a.k_one_round && rounded * a.q_parts <= 2 * a.k_shares;
    w.part = first_ones ? blk / rounded : blk / kXcds % a.q_parts;
    const int slot = first_ones ? blk % rounded : blk / (kXcds * a.q_parts) * kXcds + blk % kXcds;
    if (slot >= slots) return w;
    const int item = __builtin_amdgcn_readfirstlane(a.order ? a.order[slot] : slot);
    w.parts = a.q_parts > 1 && item >= 0 ? __builtin_amdgcn_readfirstlane(q_item_parts(a, item)) : 1;
    if (w.part >= w.parts) return w;
    w.item = item;
    w.slot0 = item * a.q_parts;
  }
  return w;
}

// F32: dK and dV (of both kinds of keys) are stored in fp32.
template <int CT, int D, bool KEYS, bool F32>
__global__ __launch_bounds__(256, D == 128 ? 2 : D == 64 ? 3 : 4) void attn_bwd_kernel(BwdArgs a, int slots) {
  using G = BwdGeom<D>;
  using S = BwdShape<D, KEYS>;
  constexpr int KS = D / 32, DT = D / 16, NA = KEYS ? 2 : 1;
  // Two pairs of tiles (Y1, Y2) and, where the columns are keys, of row values.  Arrays of their own: the compiler
  // then knows that copies into one do not touch what is read from another.
  __shared__ u32x4 lds_a[2 * S::kTile / 16], lds_b[2 * S::kTile / 16];
  __shared__ u32x4 lds_x[S::kX2Lds ? 128 * G::kRow / 16 : 1];
  __shared__ float rows_a[2 * S::kStep], rows_b[2 * S::kStep];
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, sl = lane & 15;

  const BwdItem w = bwd_item<KEYS>(a, (int)blockIdx.x, slots);
  if (w.item < 0) return;
  const int item = w.item, part = w.part, parts = w.parts;
  const bool of_pooled = w.of_pooled;
  const int ndb = (a.Nd + 127) >> 7;
  const int nob = of_pooled ? ndb : KEYS ? a.nkb : a.nqb;
  const int bh = item / nob, ob = item - bh * nob;
  const int b = bh / a.H, h = bh - b * a.H;
  const int Nown = of_pooled ? a.Nd : KEYS ? a.Nk : a.Nq;
  const Rows hq = head_rows<2>(a.q, a.qs, b, h), hdo = head_rows<2>(a.dout, a.dos, b, h);
  const Rows hk = head_rows<2>(a.k, a.ks, b, h), hv = head_rows<2>(a.v, a.vs, b, h);
  const Rows hkd = head_rows<2>(a.kd, a.kds, b, h), hvd = head_rows<2>(a.vd, a.vds, b, h);

  // This group's share [lo, hi) of the item's blocks: the listed ones, then (queries) the pooled keys'; its steps are
  // their rows, without those that would start past the end of a last block.
  constexpr int PB = 128 / S::kStep;  // steps of a block
  const int Ny = KEYS ? a.Nq : a.Nk;
  const SA_CONST int32_t* list =
      (const SA_CONST int32_t*)(KEYS ? a.kidx + (int64_t)item * a.nqb : a.idx + (int64_t)item * a.nkb);
  const int cnt = of_pooled ? a.comp_qblocks
                            : __builtin_amdgcn_readfirstlane(((const SA_CONST int32_t*)(KEYS ? a.kcounts : a.counts))[item]);
  const int blocks = cnt + (!KEYS && ob < a.comp_qblocks ? ndb : 0);
  const int lo = part_begin(blocks, part, parts), hi = part_begin(blocks, part + 1, parts);
  auto steps_to = [&](int first, int last, int n) {  // of blocks first .. last - 1, n rows in all
    return first < last ? PB * (last - first - 1) + min(PB, (n - (last - 1) * 128 + S::kStep - 1) / S::kStep) : 0;
  };
  int n1;
  if (of_pooled) {
    n1 = steps_to(lo, hi, Ny);
  } else {
    const int end = min(hi, cnt);
    n1 = lo < end ? PB * (end - lo - 1) + steps_to(list[end - 1], list[end - 1] + 1, Ny) : 0;
  }
  const int dlo = max(lo - cnt, 0), nd = KEYS ? 0 : steps_to(dlo, max(hi - cnt, 0), a.Nd);
  const int steps = n1 + nd;
  // first row of step t < steps
  auto row_of = [&](int t) __attribute__((always_inline)) {
    if (of_pooled) return lo * 128 + t * S::kStep;
    if (t >= n1) return dlo * 128 + (t - n1) * S::kStep;
    return list[lo + t / PB] * 128 + t % PB * S::kStep;
  };
  const uint32_t st1 = (uint32_t)(KEYS ? a.qs[2] : a.ks[2]) * 2, st2 = (uint32_t)(KEYS ? a.dos[2] : a.vs[2]) * 2;
  const uint32_t sd1 = (uint32_t)a.kds[2] * 2, sd2 = (uint32_t)a.vds[2] * 2;
  const BwdLanes<D> L = bwd_lanes<D>(lane);
  // A tile is NI copy instructions (kCopyRows rows each): instruction i < NI of a pair fills Y1's, the others Y2's, and
  // wave w issues w, w + 4, ...
  constexpr int NI = S::kTile / 1024;
  // this wave's share of step t into a tile pair
  auto copy = [&](int t, SA_LDS char* dst, SA_LDS char* dst_rows) __attribute__((always_inline)) {
    const int row0 = row_of(t);
    const bool pooled = !KEYS && t >= n1;
    const int valid = (pooled ? a.Nd : Ny) - row0;
    const uint32_t s1 = pooled ? sd1 : st1, s2 = pooled ? sd2 : st2;
    const char* p1 = (KEYS ? hq.base : pooled ? hkd.base : hk.base) + (int64_t)row0 * s1;
    const char* p2 = (KEYS ? hdo.base : pooled ? hvd.base : hv.base) + (int64_t)row0 * s2;
    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(p1, (uint32_t)valid * s1), r2 = make_rsrc(p2, (uint32_t)valid * s2);
#pragma unroll
    for (int j = 0; j < (2 * NI + 3) / 4; ++j) {
      const int i = 4 * j + wave, ti = i % NI;
      const bool of2 = i >= NI;
      const int row = G::kCopyRows * ti + lane / G::kChunks;
      dma16(of2 ? r2 : r1, (SA_LDS void*)(dst + i * 1024),
            (uint32_t)row * (of2 ? s2 : s1) + (uint32_t)(((lane % G::kChunks) ^ G::swz(row)) * 16));
    }
    if constexpr (KEYS) {
      // the rows' lse and -delta; the workspace has 128 rows of every q-block
      if (wave < S::kStep / 32)
        dma4(make_rsrc(a.row_vals + 2 * ((int64_t)bh * a.nqb * 128 + row0), S::kStep * 8), (SA_LDS void*)(dst_rows + wave * 256),
             (uint32_t)(wave * 256 + lane * 4));
    }
  };
  // (the first step's rows fly while the columns' operands are fetched)
  SA_LDS char *ta = (SA_LDS char*)lds_a, *tb = (SA_LDS char*)lds_b, *ra = (SA_LDS char*)rows_a, *rb = (SA_LDS char*)rows_b;
  if (steps > 0) copy(0, ta, ra);

  // the columns' operands: column 16 ct + l % 16 of the wave, d slice 32 ks + 8 (l / 16); columns past the
  // end repeat the last one (in LDS: are zero) and are not stored
  const int own0 = ob * 128 + wave * 32;
  const Rows x1 = of_pooled ? hkd : KEYS ? hk : hq, x2 = of_pooled ? hvd : KEYS ? hv : hdo;
  SA_LDS char* xt = (SA_LDS char*)lds_x + (S::kX2Lds ? wave * 32 * G::kRow : 0);
  u32x4 b1[2][KS], b2[2][KS];
  float lse2[2], ndelta[2], m[2];  // m: f16, log2 of the columns' dS factors
  if constexpr (S::kX2Lds) {
    const uint32_t st = (uint32_t)x2.stride * 2;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(x2.base + (int64_t)own0 * st, own0 < Nown ? (uint32_t)(Nown - own0) * st : 0u);
#pragma unroll
    for (int j = 0; j < 32 / G::kCopyRows; ++j) {
      const int row = G::kCopyRows * j + lane / G::kChunks;
      dma16(rs, (SA_LDS void*)(xt + j * 1024), (uint32_t)row * st + (uint32_t)(((lane % G::kChunks) ^ G::swz(row)) * 16));
    }
  }
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    lse2[ct] = ndelta[ct] = 0.f;
    m[ct] = kDsStart;
    const int own = min(own0 + 16 * ct + sl, Nown - 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      b1[ct][ks] = *(const u32x4*)(x1.base + ((int64_t)own * x1.stride + 32 * ks + 8 * g) * 2);
      if constexpr (!S::kX2Lds) b2[ct][ks] = *(const u32x4*)(x2.base + ((int64_t)own * x2.stride + 32 * ks + 8 * g) * 2);
    }
    if constexpr (!KEYS) {
      const Rows o = head_rows<2>(a.out, a.os, b, h);
      float dl = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 ov = *(const u32x4*)(o.base + ((int64_t)own * o.stride + 32 * ks + 8 * g) * 2);
#pragma unroll
        for (int e = 0; e < 8; ++e) dl += unpack16<CT>(ov[e >> 1], e & 1) * unpack16<CT>(b2[ct][ks][e >> 1], e & 1);
      }
      dl = sum_col16(dl);
      const int64_t r = (int64_t)bh * a.Nq + own;
      lse2[ct] = a.lse[r] * kLog2e;
      if (a.dlse != nullptr) dl -= a.dlse[r];
      // a row without keys has no gradient; neither have rows past the end
      if (own0 + 16 * ct + sl >= a.Nq) lse2[ct] = pos_inf();
      ndelta[ct] = lse2[ct] == pos_inf() ? 0.f : -dl;
      if (g == 0 && part == 0) {
        const int64_t at = row_slot((int64_t)bh * a.nqb * 128 + own0 + 16 * ct + sl);
        a.row_vals[at] = lse2[ct];
        a.row_vals[at + 4] = ndelta[ct];
      }
    }
  }
  f32x4 acc[NA][DT][2];
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[n][dt][0] = acc[n][dt][1] = f32x4{};
  const float c2 = a.scale * kLog2e;
  // times c2: -inf, a weight of 0 (a scale of 0 makes dQ 0 whatever the weight)
  const float gone = c2 > 0.f ? neg_inf() : c2 < 0.f ? pos_inf() : 0.f;
  // What S starts at: 0, or `gone` for keys that do not exist (rows of queries that do not have an lse of +inf).  Set
  // where such rows begin and end: with a comparison for each row of every step, the dQ kernel took 7% longer at D = 128
  // (12 heads of 32760 tokens: 1.62 -> 1.51 ms).
  f32x4 start[2] = {f32x4{}, f32x4{}};
  bool short_rows = false;

  auto step = [&](int t, SA_LDS char* y1, SA_LDS char* rows, SA_LDS char* next, SA_LDS char* next_rows) __attribute__((always_inline)) {
    const bool pooled = of_pooled || t >= n1;
    if (t + 1 < steps) copy(t + 1, next, next_rows);
    const int left = (!KEYS && pooled ? a.Nd : Ny) - row_of(t);  // streamed rows that exist
    const float bias = pooled ? a.comp_bias : 0.f;
    if constexpr (KEYS)
      repeat_last_row<S::kStep, G::kChunks>(y1, left, tid, [](int row, int ch) { return row * G::kRow + (ch ^ G::swz(row)) * 16; });
    // (unrolled, so that the reads' addresses are constants: 1.60 -> 1.56 ms for dQ of the same, 259 -> 250 us at D = 64)
#pragma unroll
    for (int sub = 0; sub < S::kStep / 32 && 32 * sub < left; ++sub) {
      if (!KEYS && (left - 32 * sub < 32 || short_rows)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) start[i >> 2][i & 3] = 32 * sub + 16 * (i >> 2) + 4 * g + (i & 3) < left ? 0.f : gone;
        short_rows = left - 32 * sub < 32;
      }
      bwd_rows32<CT, D, KEYS>(y1, (uint32_t)(32 * sub * G::kRow), rows + 256 * sub, xt, L, b1, b2, acc, lse2, ndelta, m, bias, c2,
                              start, g);
    }
    drain_then_barrier();  // the next step's rows have landed, every wave is done with this one's
  };

  drain_then_barrier();
  for (int t = 0; t < steps; t += 2) {
    step(t, ta, ra, tb, rb);
    if (t + 1 < steps) step(t + 1, tb, rb, ta, ra);
  }

  float f0[2], f1[2];
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    f0[ct] = CT == kF16 ? a.scale * fast_exp2(-m[ct]) : a.scale;
    f1[ct] = CT == kF16 ? fast_exp2(-kPShift) : 1.f;
  }
  if (parts > 1) {
    // the part's fp32 sums as the registers hold them, 1 KB per instruction
    float* to = (KEYS ? a.part_k : a.part_q) + (int64_t)(w.slot0 + part) * NA * 128 * D + wave * 32 * D + lane * 4;
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
          *reinterpret_cast<f32x4*>(to + n * 128 * D + ct * 16 * D + dt * 256) = acc[n][dt][ct] * (n ? f1 : f0)[ct];
    return;
  }
  // every wave through a part of its own of what is free now
  SA_LDS char* buf = S::kX2Lds ? xt : (wave < 2 ? ta : tb) + (wave & 1) * 64 * D;
  if constexpr (!KEYS) {
    const Rows o = head_rows<2>(a.dq, a.dqs, b, h);
    store_columns<CT, D>(const_cast<char*>(o.base), o.stride, own0, Nown, acc[0], f0, buf, lane);
  } else if constexpr (F32) {
    const Rows ok = of_pooled ? head_rows<4>(a.dkd, a.dkds, b, h) : head_rows<4>(a.dk, a.dks, b, h);
    const Rows ov = of_pooled ? head_rows<4>(a.dvd, a.dvds, b, h) : head_rows<4>(a.dv, a.dvs, b, h);
    store_columns_f32<D>(const_cast<char*>(ok.base), ok.stride, own0, Nown, acc[0], f0, lane);
    store_columns_f32<D>(const_cast<char*>(ov.base), ov.stride, own0, Nown, acc[NA - 1], f1, lane);
  } else {
    const Rows ok = of_pooled ? head_rows<2>(a.dkd, a.dkds, b, h) : head_rows<2>(a.dk, a.dks, b, h);
    const Rows ov = of_pooled ? head_rows<2>(a.dvd, a.dvds, b, h) : head_rows<2>(a.dv, a.dvs, b, h);
    store_columns<CT, D>(const_cast<char*>(ok.base), ok.stride, own0, Nown, acc[0], f0, buf, lane);
    store_columns<CT, D>(const_cast<char*>(ov.base), ov.stride, own0, Nown, acc[NA - 1], f1, buf, lane);
  }
}

// The parts' sums added in order, rounded and stored.  A unit is 16 columns of one result of a cut list (dK or dV of a
// key block, dQ of a query block with q_parts > 1), added as the parts' registers hold them, the loads of several
// parts in flight.  Bound by latency, 4 us without a cut list, and by the traffic: 62 us for the fp32 call's 1536 query
// parts and its cut key lists, 14 us for an image with a prompt (30 heads of 9 blocks).
constexpr int kJoinGroups = 1024;

template <int CT, int D>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(BwdArgs a) {
  constexpr int ES = ElemSize<CT>::value;
  constexpr int DT = D / 16, UNROLL = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nsparse = a.B * a.H * a.nkb, ndb = (a.Nd + 127) >> 7;
  const int key_units = a.k_slots > 0 ? a.cut_slot[0] * 16 : 0;
  const int units = key_units + (a.q_parts > 1 ? a.B * a.H * a.nqb * 8 : 0);
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const bool of_keys = unit < key_units;
    const int r16 = unit & 7, n = of_keys ? (unit >> 3) & 1 : 0;
    const int slot = of_keys ? a.cut_slot[1 + (unit >> 4)] : ((unit - key_units) >> 3) * a.q_parts;
    const int item = of_keys ? a.slot_item[slot] : (unit - key_units) >> 3;
    const int parts = of_keys ? a.slot_part[slot] >> 16 : q_item_parts(a, item);
    if (parts < 2) continue;  // stored whole
    const bool of_pooled = of_keys && item >= nsparse;
    const int it = of_pooled ? item - nsparse : item, nob = of_pooled ? ndb : of_keys ? a.nkb : a.nqb;
    const int bh = it / nob, ob = it - bh * nob, b = bh / a.H, h = bh - b * a.H;
    const int Nown = of_pooled ? a.Nd : of_keys ? a.Nk : a.Nq;
    const bool f32 = of_keys && a.f32_key_grads;
    const int es = f32 ? 4 : ES;
    auto rows = [&](void* p, const int64_t (&st)[4]) { return Rows{(char*)p + ((int64_t)b * st[0] + (int64_t)h * st[1]) * es, st[2]}; };
    const Rows o = !of_keys ? rows(a.dq, a.dqs)
                   : of_pooled ? (n ? rows(a.dvd, a.dvds) : rows(a.dkd, a.dkds))
                               : (n ? rows(a.dv, a.dvs) : rows(a.dk, a.dks));
    const int64_t per = (int64_t)(of_keys ? 2 : 1) * 128 * D;  // floats of a part
    const float* from = (of_keys ? a.part_k : a.part_q) + (int64_t)slot * per + n * 128 * D + r16 * 16 * D + lane * 4;
    const int own = ob * 128 + r16 * 16 + (lane & 15);
    for (int dt = wave; dt < DT; dt += 4) {
      f32x4 sum = f32x4{};
      for (int p = 0; p < parts; p += UNROLL) {
        f32x4 x[UNROLL];
#pragma unroll
        for (int e = 0; e < UNROLL; ++e)
          x[e] = p + e < parts ? *reinterpret_cast<const f32x4*>(from + (p + e) * per + dt * 256) : f32x4{};
#pragma unroll
        for (int e = 0; e < UNROLL; ++e) sum += x[e];
      }
      if (own >= Nown) continue;
      char* to = const_cast<char*>(o.base) + ((int64_t)own * o.stride + 16 * dt + 4 * (lane >> 4)) * es;
      if (f32) store4<kF32>(to, sum[0], sum[1], sum[2], sum[3]);
      else store4<CT>(to, sum[0], sum[1], sum[2], sum[3]);
    }
  }
}

// ------------------------------------------------------------------------------------
// fp32 operands, on fp32 matrix instructions (16x16x4: exact products, fp32 sums; a split into bf16 pairs, as
// the forward's, would leave the gradients at 16 bits).  A wave owns 16 columns, a group 64 (half of a block),
// and streams 32 rows per step through two pairs of LDS tiles.  Contraction step (c, e) of S and dP takes
// d = 16 c + 4 g + e of lane group g, four steps per 16-byte read; step i of the other products takes
// streamed row 4 g + i, the row of accumulator register i, one 4-byte read per 16 columns d.  Chunks
// are swizzled by row & 7: neither read has bank conflicts.  Bound by the matrix cores, busy 93%
// of the time that a CU has work: 12 heads of 4096 tokens, 74%, D = 128 take 0.93 + 1.27 ms, 0.13 PFLOP/s of the seven
// products where the library's 8192^3 reaches 0.153 (D = 64 0.49 + 0.59, D = 32 0.27 + 0.30); the rest is the uneven end of lists of 12 to 32 tiles.
// ------------------------------------------------------------------------------------
template <int D, bool KEYS>
__global__ __launch_bounds__(256, KEYS ? 2 : 3) void attn_bwd_f32_kernel(BwdArgs a, int slots) {
  constexpr int C4 = D / 16, DT = D / 16, NA = KEYS ? 2 : 1;
  // Streamed rows of a step, steps of a block: short steps of dQ at D = 128 leave room for a third group (1.10 -> 1.06 ms).
  constexpr int STEP = !KEYS && D == 128 ? 16 : 32, PB = 128 / STEP;
  constexpr int kRow = 4 * D, kTile = STEP * kRow, kChunks = D / 4;
  __shared__ u32x4 lds_a[2 * kTile / 16], lds_b[2 * kTile / 16];
  __shared__ float rows_a[64], rows_b[64];  // KEYS: lse and -delta, as in the workspace
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, sl = lane & 15;
  // the two halves of a block run on one XCD, one after the other
  const int half = (int)(blockIdx.x / kXcds) & 1;
  const int blk = (int)(blockIdx.x / (2 * kXcds)) * kXcds + (int)(blockIdx.x % kXcds);
  if (!KEYS && blk == 0 && half == 1) return;  // (half 0 plans)
  const BwdItem w = bwd_item<KEYS>(a, blk, slots);
  if (w.item < 0) return;
  const int item = w.item, nob = KEYS ? a.nkb : a.nqb;
  const int bh = item / nob, ob = item - bh * nob;
  const int b = bh / a.H, h = bh - b * a.H;
  const int Nown = KEYS ? a.Nk : a.Nq, Ny = KEYS ? a.Nq : a.Nk;
  const int own0 = ob * 128 + half * 64 + wave * 16, own = own0 + sl, own_c = min(own, Nown - 1);
  const Rows hq = head_rows<4>(a.q, a.qs, b, h), hdo = head_rows<4>(a.dout, a.dos, b, h);
  const Rows hk = head_rows<4>(a.k, a.ks, b, h), hv = head_rows<4>(a.v, a.vs, b, h);
  const Rows x1 = KEYS ? hk : hq, x2 = KEYS ? hv : hdo;  // columns
  const Rows y1 = KEYS ? hq : hk, y2 = KEYS ? hdo : hv;  // streamed
  f32x4 b1[C4], b2[C4];
#pragma unroll
  for (int c = 0; c < C4; ++c) {
    b1[c] = *(const f32x4*)(x1.base + ((int64_t)own_c * x1.stride + 16 * c + 4 * g) * 4);
    b2[c] = *(const f32x4*)(x2.base + ((int64_t)own_c * x2.stride + 16 * c + 4 * g) * 4);
  }
  float lse2 = 0.f, ndelta = 0.f;  // of the owned query
  if constexpr (!KEYS) {
    const Rows o = head_rows<4>(a.out, a.os, b, h);
    float dl = 0.f;
#pragma unroll
    for (int c = 0; c < C4; ++c) {
      const f32x4 x = *(const f32x4*)(o.base + ((int64_t)own_c * o.stride + 16 * c + 4 * g) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) dl += x[e] * b2[c][e];
    }
    dl = sum_col16(dl);
    const int64_t r = (int64_t)bh * a.Nq + own_c;
    lse2 = a.lse[r] * kLog2e;
    if (a.dlse != nullptr) dl -= a.dlse[r];
    // a row without keys has no gradient; neither have rows past the end
    if (own >= a.Nq) lse2 = pos_inf();
    ndelta = lse2 == pos_inf() ? 0.f : -dl;
    if (g == 0 && w.part == 0) {
      const int64_t at = row_slot((int64_t)bh * a.nqb * 128 + own);
      a.row_vals[at] = lse2;
      a.row_vals[at + 4] = ndelta;
    }
  }
  f32x4 acc[NA][DT];
#pragma unroll
  for (int n = 0; n < NA; ++n)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[n][dt] = f32x4{};
  const float c2 = a.scale * kLog2e;
  const float gone = c2 > 0.f ? neg_inf() : c2 < 0.f ? pos_inf() : 0.f;  // as in the 16-bit kernel

  const SA_CONST int32_t* list =
      (const SA_CONST int32_t*)(KEYS ? a.kidx + (int64_t)item * a.nqb : a.idx + (int64_t)item * a.nkb);
  const int cnt = __builtin_amdgcn_readfirstlane(((const SA_CONST int32_t*)(KEYS ? a.kcounts : a.counts))[item]);
  const int lo = part_begin(cnt, w.part, w.parts), hi = part_begin(cnt, w.part + 1, w.parts);
  const int steps = own0 - wave * 16 < Nown && lo < hi ? PB * (hi - lo - 1) + min(PB, (Ny - list[hi - 1] * 128 + STEP - 1) / STEP) : 0;
  const uint32_t st1 = (uint32_t)y1.stride * 4, st2 = (uint32_t)y2.stride * 4;
  auto copy = [&](int t, SA_LDS char* dst, SA_LDS char* dst_rows) __attribute__((always_inline)) {
    const int row0 = list[lo + t / PB] * 128 + t % PB * STEP;
    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(y1.base + (int64_t)row0 * st1, (uint32_t)(Ny - row0) * st1);
    const __amdgpu_buffer_rsrc_t r2 = make_rsrc(y2.base + (int64_t)row0 * st2, (uint32_t)(Ny - row0) * st2);
    constexpr int NI = kTile / 1024;  // copy instructions of a tile, dealt to the waves
#pragma unroll
    for (int j = 0; j < NI / 4; ++j) {
      const int i = 4 * j + wave, at = i * 64 + lane, row = at / kChunks, ch = at % kChunks ^ (row & 7);
      dma16(r1, (SA_LDS void*)(dst + i * 1024), (uint32_t)row * st1 + (uint32_t)(ch * 16));
      dma16(r2, (SA_LDS void*)(dst + kTile + i * 1024), (uint32_t)row * st2 + (uint32_t)(ch * 16));
    }
    if (KEYS && wave == 0)
      dma4(make_rsrc(a.row_vals + 2 * ((int64_t)bh * a.nqb * 128 + row0), 256), (SA_LDS void*)dst_rows, (uint32_t)(lane * 4));
  };
  // Lane offsets in a tile: row reads of even and odd c (row l % 16, chunk 4 c + g), and the 4-byte reads of row
  // 4 g + i at even and odd dt (column 16 dt + l % 16); the rest of c and dt moves whole 128 bytes.
  uint32_t row_at[2], col_at[4][2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    row_at[p] = (uint32_t)(sl * kRow + ((4 * p + g) ^ (sl & 7)) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) col_at[i][p] = (uint32_t)(4 * g * kRow + (((4 * p + (sl >> 2)) ^ ((4 * g + i) & 7)) * 16) + (sl & 3) * 4);
  }
  auto step = [&](int t, SA_LDS char* tile, SA_LDS char* rows, SA_LDS char* next, SA_LDS char* next_rows) __attribute__((always_inline)) {
    if (t + 1 < steps) copy(t + 1, next, next_rows);
    const int left = Ny - (list[lo + t / PB] * 128 + t % PB * STEP);
    if constexpr (KEYS)
      repeat_last_row<32, kChunks>(tile, left, tid, [](int row, int ch) { return row * kRow + (ch ^ (row & 7)) * 16; });
#pragma unroll 1
    for (int rt = 0; rt < STEP / 16; ++rt) {
      f32x4 s = f32x4{}, u = f32x4{ndelta, ndelta, ndelta, ndelta}, rl = f32x4{lse2, lse2, lse2, lse2};
      if constexpr (KEYS) {
        rl = *(SA_LDS const f32x4*)(rows + (4 * rt + g) * 32);
        u = *(SA_LDS const f32x4*)(rows + (4 * rt + g) * 32 + 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = 16 * rt + 4 * g + i < left ? 0.f : gone;
      }
      constexpr int AHEAD = 4, N1 = 2 * C4;  // row reads, a chunk of Y1 and of Y2 in turn
      f32x4 r[N1];
      auto read = [&](int j) { return *(SA_LDS const f32x4*)(tile + row_at[j / 2 & 1] + (j & 1) * kTile + 16 * rt * kRow + (j / 4) * 128); };
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) r[j] = read(j);
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD + (KEYS ? 2 : 0), 0);
#pragma unroll
      for (int j = 0; j < N1; ++j) {
        if (j + AHEAD < N1) {
          r[j + AHEAD] = read(j + AHEAD);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if ((j & 1) == 0) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(r[j - 1][e], b1[j / 2][e], s, 0, 0, 0);
          u = __builtin_amdgcn_mfma_f32_16x16x4f32(r[j][e], b2[j / 2][e], u, 0, 0, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      constexpr int TAHEAD = 6, N2 = 4 * DT * NA;  // 4-byte reads, row by row
      float v[N2];
      auto vread = [&](int j) {
        const int i = j / (DT * NA), dt = j / NA % DT, n = j % NA;
        return *(SA_LDS const float*)(tile + col_at[i][dt & 1] + n * kTile + (16 * rt + i) * kRow + (dt >> 1) * 128);
      };
#pragma unroll
      for (int j = 0; j < TAHEAD; ++j) v[j] = vread(j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = fast_exp2(__builtin_fmaf(s[i], c2, -rl[i]));
        u[i] *= s[i];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < N2; ++j) {
        const int i = j / (DT * NA), dt = j / NA % DT, n = j % NA;
        if (j + TAHEAD < N2) {
          v[j + TAHEAD] = vread(j + TAHEAD);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        acc[n][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], n ? s[i] : u[i], acc[n][dt], 0, 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    drain_then_barrier();  // the next step's rows have landed, every wave is done with this one's
  };
  SA_LDS char *ta = (SA_LDS char*)lds_a, *tb = (SA_LDS char*)lds_b, *ra = (SA_LDS char*)rows_a, *rb = (SA_LDS char*)rows_b;
  if (steps > 0) copy(0, ta, ra);
  drain_then_barrier();
  for (int t = 0; t < steps; t += 2) {
    step(t, ta, ra, tb, rb);
    if (t + 1 < steps) step(t + 1, tb, rb, ta, ra);
  }

  if (w.parts > 1) {
    float* to = (KEYS ? a.part_k : a.part_q) + (int64_t)(w.slot0 + w.part) * NA * 128 * D + (half * 4 + wave) * 16 * D + lane * 4;
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + n * 128 * D + dt * 256) = acc[n][dt] * (n ? 1.f : a.scale);
    return;
  }
  if (own >= Nown) return;
#pragma unroll
  for (int n = 0; n < NA; ++n) {
    const Rows o = !KEYS ? head_rows<4>(a.dq, a.dqs, b, h) : n ? head_rows<4>(a.dv, a.dvs, b, h) : head_rows<4>(a.dk, a.dks, b, h);
    float* to = (float*)const_cast<char*>(o.base) + (int64_t)own * o.stride + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + 16 * dt) = acc[n][dt] * (n ? 1.f : a.scale);
  }
}

// Blocks of the rounds that fp32 lists are cut for: four of three groups per CU at D = 128, two of four below.
static int64_t f32_round_blocks(int D) { return (D == 128 ? 12 : 8) * (int64_t)device_cu_count() / 2; }

// Parts of the lists: see BwdArgs.  Query blocks are cut where all of them are fewer than the groups that run at a
// time; the sizes allow for every smaller call's cuts, so that a workspace serves those too.
size_t block_sparse_bwd_workspace(BwdArgs& a, int dtype, int D, void* workspace) {
  const int64_t nbh = (int64_t)a.B * a.H, ndb = (a.Nd + 127) / 128, rows = nbh * a.nqb, items = nbh * (a.nkb + ndb);
  // that run at a time
  const int64_t groups = (D == 128 ? 2 : D == 64 && dtype != kF32 ? 3 : 4) * device_cu_count();
  const int64_t qlist = a.nkb + ndb > 1 ? a.nkb + ndb : 1;
  // 16-bit: as many parts as run at once, or barely do not.  Where every list's blocks would not as parts of their own, parts
  // have four blocks if lists allow (30 heads of 9 q-blocks with 2.3 tiles each and one of pooled keys: 44 -> 35 us; whole calls
  // with at most one, two, four and eight: [1,24,1000] 70, 63, 62 and 62 us, [1,40,1101] 95, 93, 88 and 85, [1,12,2048] 85,
  // 85, 80 and 84, [1,4,8000] 119, 119, 117 and 109, [1,12,2000] with pooled keys 81, 79, 76 and 79).
  // fp32 (a block is two groups, and its blocks' products outweigh a part's sums by far): some rounds, for an even end.
  int64_t q_parts = rows > 0 && rows < groups ? (groups + rows - 1) / rows : 1;
  const int64_t dense_share = (rows * qlist + groups - 1) / groups;
  a.q_share = dtype == kF32 || dense_share < 1 ? 1 : dense_share < 4 ? (int)dense_share : 4;
  const int64_t q_groups = f32_round_blocks(D);
  if (dtype == kF32) q_parts = rows > 0 && rows < q_groups ? (q_groups + rows - 1) / rows : 1;
  q_parts = q_parts < qlist ? q_parts : qlist;
  a.k_one_round = dtype != kF32;
  a.k_shares = (int)(dtype == kF32 ? 2 * groups : groups);  // fp32: of four rounds too (1.41 -> 1.27 ms)
  const int64_t all = items * a.nqb, most = 2 * (int64_t)a.k_shares;
  const int64_t k_slots = a.nqb < 2 ? 0 : all < most ? all : most;
  const int64_t q_most = 2 * (dtype == kF32 ? q_groups : groups), q_slots = rows * qlist < q_most ? rows * qlist : q_most;
  a.q_parts = (int)q_parts;
  a.k_slots = (int)((k_slots + kXcds - 1) / kXcds * kXcds);
  char* p = (char*)workspace;
  auto take = [&](int64_t bytes) {
    char* at = p;
    p += (bytes + 255) / 256 * 256;
    return at;
  };
  a.row_vals = (float*)take(rows * 128 * 8);
  a.part_q = (float*)take(q_slots * 128 * D * 4);
  a.part_k = (float*)take(a.k_slots * 2 * 128 * (int64_t)D * 4);
  a.split_base = (int32_t*)take(items * 4);
  a.slot_item = (int32_t*)take(a.k_slots * 4);
  a.slot_part = (int32_t*)take(a.k_slots * 4);
  a.extra_slot = (int32_t*)take(a.k_slots * 4);
  a.cut_slot = (int32_t*)take((2 + a.k_slots) * 4);
  return (size_t)(p - (char*)workspace);
}

template <int CT, int D>
static hipError_t launch_bwd_d(const BwdArgs& args, int qgrid, int kgrid, hipStream_t stream) {
  BwdArgs a = args;
  hipError_t e = hipSuccess;
  auto up = [](int n) { return (n + kXcds - 1) / kXcds * kXcds; };
  if (qgrid > 0) {
    const int groups = kXcds + up(qgrid) * a.q_parts;
    if constexpr (CT == kF32) attn_bwd_f32_kernel<D, false><<<2 * groups, 256, 0, stream>>>(a, qgrid);
    else attn_bwd_kernel<CT, D, false, false><<<groups, 256, 0, stream>>>(a, qgrid);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  } else {
    a.k_slots = 0;  // nothing was planned
  }
  const int groups = a.k_slots + up(a.B * a.H * ((a.Nd + 127) / 128)) + up(kgrid);
  if (groups > 0) {
    if constexpr (CT == kF32) attn_bwd_f32_kernel<D, true><<<2 * groups, 256, 0, stream>>>(a, kgrid);
    else if (D == 128 && a.f32_key_grads) attn_bwd_kernel<CT, D, true, D == 128><<<groups, 256, 0, stream>>>(a, kgrid);
    else attn_bwd_kernel<CT, D, true, false><<<groups, 256, 0, stream>>>(a, kgrid);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  // (a cut list has two slots at least)
  const int64_t joins = (int64_t)a.k_slots / 2 * 16 + (a.q_parts > 1 ? (int64_t)a.B * a.H * a.nqb * 8 : 0);
  if (joins > 0) attn_bwd_join_kernel<CT, D><<<(int)(joins < kJoinGroups ? joins : kJoinGroups), 256, 0, stream>>>(a);
  return hipGetLastError();
}

template <int CT>
static hipError_t launch_bwd_dt(const BwdArgs& args, int D, hipStream_t stream) {
  BwdArgs a = args;
  const int nbh = a.B * a.H;
  // The orders keep a head's blocks on one XCD, for its L2, which leaves the XCDs with unlike work where heads are few and
  // unlike.  fp32 products take so long that the reads matter less: with fewer than two heads for an XCD the plain order is
  // faster (heads of densities of their own, whole calls in us, plan's -> plain order, D = 128: [1,8,4096] 1109 -> 1053,
  // [1,10,4096] 1055 -> 955, [1,12,4096] 1529 -> 1471, [1,4,9000] 1764 -> 1627, [1,12,17000] 9042 -> 8480, [1,8,30000] 15002 ->
  // 10440; the same at D = 64 and 32; six heads of 4096 lose 1%), with more the plan's (plain -> plan's: [1,16,4096] 1661 -> 1631,
  // [1,18,4096] 1861 -> 1789, [1,32,4096] 4000 -> 3620, [1,24,7680] 4483 -> 4357, D = 64 [1,20,4096] 1117 -> 1066).
  if (CT == kF32 && nbh < 2 * kXcds) a.order = a.korder = nullptr;
  const int qgrid = a.order ? plan_launch_slots(nbh * a.nqb, a.nqb) : nbh * a.nqb;
  const int kgrid = a.korder ? plan_launch_slots(nbh * a.nkb, a.nkb) : nbh * a.nkb;
  if (D == 128) return launch_bwd_d<CT, 128>(a, qgrid, kgrid, stream);
  if (D == 64) return launch_bwd_d<CT, 64>(a, qgrid, kgrid, stream);
  return launch_bwd_d<CT, 32>(a, qgrid, kgrid, stream);
}

hipError_t launch_block_sparse_bwd(const BwdArgs& a, int dtype, int D, hipStream_t stream) {
  if (dtype == kBF16) return launch_bwd_dt<kBF16>(a, D, stream);
  if (dtype == kF16) return launch_bwd_dt<kF16>(a, D, stream);
  return launch_bwd_dt<kF32>(a, D, stream);
}

}  // namespace sa
