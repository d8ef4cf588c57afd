// Attention over the paged 8-bit cache for many rows per sequence (prompts and chunks of them): tcgen05.
//
// An item is 128 NG rows of q (tokens x heads of one kv head's group) of a sequence and kv head; its tiles are 64 tokens.
// NG = 1: two CTAs share an SM; NG = 2, for 256 rows and more: one CTA, whose two groups of 128 rows share the expanded codes.
//   S = Q K^T     M = 128 rows, N = 64 tokens:  Q and the tile's keys in shared memory, S in tensor memory (two buffers)
//   P             softmax warps read S (one row per thread), write p as f16 over it
//   O += P V      M = 128 rows, N = DW channels: P out of tensor memory, the tile's values [channel][token] in shared memory
// The codes become f16 whole numbers (exact); q is f16 after a power of two per row (exact for f16, and for bf16 down to
// 2^-24 of the row's largest element).  Scales meet fp32 numbers: the keys' in the scores, the values' in the exponent,
//   p' = 2^(score + log2(v_scale) - reference),
// so that p' is rounded once, and finest where p v_scale is largest, whatever the scales of the pages are.  The row's reference is
// raised only when score + log2(v_scale) passes it by 12 (p' then stays below 2^12), O is rescaled then, by the row's thread.
// The sum of exponentials has a reference of its own, the running maximum of the scores: it takes p' before the rounding, 64 of
// them at a time, times 2^(reference - log2(v_scale) - maximum) (two units of 2^-23 off at most, as 2^x is).
//
// Per tile and 128 rows: 512 tensor clocks (DW = 128), 8192 exponentials (512 clocks of the special function unit).  While one
// group's (or CTA's) softmax warps work, the other's products run.
//
// Roles: warps 0 .. 4 NG - 1 softmax, then one warp for bulk copies of the raw codes (ring of four units), one that issues the MMAs,
// two (NG = 2: one) that turn the keys' codes into an operand, as many for the values' (128-byte swizzle; [token][64 channels]
// twice, [channel][64 tokens]).  With NG = 1 a row's 64 scores are read twice, 32 at a time, which keeps a thread below 96 registers.
// All warps write the outputs, by way of shared memory, so that rows go out whole.
// The work is cut into equal ranges as in kv_attend.cu, with the same slices and tickets.  Waits are bounded: a row whose
// wait ran out becomes NaN.
#include "kv_attend.cuh"
#include "trace.cuh"
#include <algorithm>
#include <cstring>

// measurement builds, per CTA: 0 entry, 1 range known, 2 first piece's q staged, 3 its tiles done, 4 last piece's tiles done, 5 exit,
// 6 tiles of the CTA
JGQ_TRACE_DEFINE(prompt, 8 * 1024)
#define PTRACE(i) JGQ_TRACE_CTA(prompt, i, 1024)

namespace jgq {

// 10 warps, or 12: three per scheduler, which leaves a thread 168 registers
constexpr int kp_threads(int ng) { return ng == 1 ? 320 : 384; }
constexpr int KP_COST = 9;                             // what an item takes beside its tiles, in tiles (see kv_attend.cu)
constexpr int KP_RAW = 4;                              // raw units (keys or values of a tile) in the ring
constexpr int KP_TMEM = 256;                           // columns per group: S and P 2 x 64, O DW
constexpr float KP_LAZY = 12.f;                        // log2 by which p v_scale may pass its row's reference
constexpr float KP_FAINT = 60.f;                       // log2 below which it is as good as nothing beside the reference

__host__ __device__ constexpr int kp_unit(int dw) { return 64 * dw; }
// q, NG buffers of expanded keys and of values, the ring; the outputs of 128 rows take their place at the end of a piece
__host__ __device__ constexpr int kp_operands(int dw, int ng) { return 128 * ng * dw * 2 + 2 * ng * 64 * dw * 2 + KP_RAW * kp_unit(dw); }
__host__ __device__ constexpr int kp_smem(int dw, int ng) { return 1024 + 1024 + kp_operands(dw, ng); }

// D[tmem] (+)= A[tmem] B[smem], f16
__device__ __forceinline__ void mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// two codes as f16 whole numbers; the values' are masked and signed
__device__ __forceinline__ uint32_t code_pair_f16(uint32_t w, uint32_t sel) {
  uint32_t r = __byte_perm(w, 0x64646464u, sel);       // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__float2half_rn(1152.f)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename XT, int DW, int NG>
__global__ void __launch_bounds__(kp_threads(NG), NG == 1 ? 2 : 1)
kv_prompt_kernel(const AttendParams p) {
  using namespace umma;
  constexpr int KP_THREADS = NG == 1 ? 320 : 384, KP_ROWS = 128 * NG, WARPS = KP_THREADS / 32;
  constexpr int UNIT = kp_unit(DW), KB = DW / 64;      // 64-channel blocks of a row
  constexpr int W_COPY = 4 * NG, W_MMA = W_COPY + 1, W_EXPAND = W_COPY + 2;
  constexpr int EW = (WARPS - W_EXPAND) / 2;           // warps per operand
  constexpr int OST = DW + 4;                          // floats per row of staged outputs
  static_assert(128 * OST * 4 <= kp_operands(DW, NG), "the outputs of 128 rows fit the operands' place");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base);
  uint64_t* raw_full = bars, *raw_empty = bars + KP_RAW;
  uint64_t *k_full = bars + 2 * KP_RAW, *k_empty = k_full + NG, *v_full = k_empty + NG, *v_empty = v_full + NG;       // per buffer
  uint64_t *s_full = v_empty + NG, *p_full = s_full + 2 * NG, *o_done = p_full + 2 * NG;         // per group, for even and odd tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2 * NG);
  uint8_t* q_smem = base + 1024;                       // [NG][KB][128 rows][128 bytes], swizzled
  uint8_t* k_smem = q_smem + KP_ROWS * DW * 2;         // [NG buffers][KB][64 tokens][128 bytes]
  uint8_t* v_smem = k_smem + NG * 64 * DW * 2;         // [NG buffers][DW channels][128 bytes]
  uint8_t* raw = v_smem + NG * 64 * DW * 2;
  float* staged = reinterpret_cast<float*>(q_smem);
  __shared__ int64_t s_pre[KP_THREADS + 1];
  __shared__ int64_t s_found[2];
  __shared__ float s_factor[KP_ROWS];                  // of a row's scores
  __shared__ float2 s_ml[KP_ROWS];                     // a row's maximum and sum, when its piece is done,
  __shared__ float s_inv[KP_ROWS];                     // what its outputs are multiplied by,
  __shared__ int64_t s_row[KP_ROWS];                   // and where they go
  __shared__ int s_flag, s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &s_abort;
  PTRACE(0);
  if (tid == 0) {
    for (int i = 0; i < KP_RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], EW); }
    for (int i = 0; i < NG; ++i) { mbar_init(&k_full[i], EW); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], EW); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < 2 * NG; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1); }
    s_abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  attend_zero_rest<XT, KP_THREADS>(p);
  AttendRange rg = attend_range<KP_ROWS, KP_COST, KP_THREADS>(p, 2 * KP_COST, s_pre, s_found);
  if ((int)blockIdx.x >= rg.G) return;
  PTRACE(1);
  if (warp == W_MMA) {
    tmem_alloc(tmem_slot, NG * KP_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int page_shift = p.P == 64 ? 0 : p.P == 128 ? 1 : 2;
  uint32_t done = 0;                                   // tiles of earlier pieces: every role's barriers count on from them
  bool ok = true;

  constexpr bool KEEP = NG == 2;
  AttendCursor<KP_ROWS, KP_COST> cursor;
  cursor.find(p, rg);
  for (int64_t idx = rg.begin; idx < rg.end; cursor.next(p, rg)) {
    const AttendPiece pc = cursor.piece(p, rg, idx);
    if (pc.t_last <= pc.t_first) break;                // the item's tiles begin behind this range
    const int n = pc.n, L = pc.L, h = pc.h;
    const int seen_item = max(0, L - n + (pc.c0 + pc.rows - 1) / p.group + 1);
    const int t_end = min(pc.t_last, (seen_item + KV_TILE - 1) / KV_TILE);
    const int nt = max(0, t_end - pc.t_first);         // tiles of this piece
    const int32_t* row_of_table = p.table + (int64_t)rg.r * p.table_stride;
    auto block_of = [&](int tile, bool& bad) {         // page and head of a tile
      const int page = row_of_table[tile >> page_shift];
      bad = page < 0 || page >= p.pages;
      return (int64_t)(bad ? 0 : page) * p.Hkv + h;
    };

    // ---- q into shared memory: a warp per row, all of a warp's rows requested at once ----
    {
      constexpr int CPL = DW / 32, QR = (KP_ROWS + WARPS - 1) / WARPS;         // channels per lane, rows per warp
      const float sign = p.scale < 0.f ? -1.f : 1.f;   // the factor of the scores is positive: a row's maximum is that of its products
      const int d0 = lane * CPL;
      using V = typename std::conditional<CPL == 4, uint2, uint32_t>::type;
      V raw_q[QR];
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        const int row = warp + r * WARPS, gr = pc.c0 + row, i = p.group == 1 ? gr : gr / p.group;
        const bool live = row < pc.rows;
        const XT* src = reinterpret_cast<const XT*>(p.q) + (live ? (int64_t)(pc.row_first + i) * p.q_token + (int64_t)(h * p.group + gr - i * p.group) * p.q_head : 0);
        raw_q[r] = V{};
        if (live && p.vec_q && d0 + CPL <= p.D) {
          raw_q[r] = *reinterpret_cast<const V*>(src + d0);
        } else if (live) {
          XT e[CPL];
#pragma unroll
          for (int j = 0; j < CPL; ++j) e[j] = d0 + j < p.D ? src[d0 + j] : from_f32<XT>(0.f);
          raw_q[r] = *reinterpret_cast<const V*>(e);
        }
      }
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        const int row = warp + r * WARPS;
        const XT* e = reinterpret_cast<const XT*>(&raw_q[r]);
        uint32_t w[CPL / 2];
        float down = 1.f;
        if constexpr (std::is_same<XT, __half>::value) {
#pragma unroll
          for (int j = 0; j < CPL / 2; ++j) w[j] = reinterpret_cast<const uint32_t*>(&raw_q[r])[j] ^ (sign < 0.f ? 0x80008000u : 0u);
        } else {
          // a power of two brings the row's largest element to [2^13, 2^14): f16 then holds what bf16 says down to 2^-27 of it
          float big = 0.f;
#pragma unroll
          for (int j = 0; j < CPL; ++j) big = fmaxf(big, fabsf(to_f32<XT>(e[j])));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
          const uint32_t x = min(max(__float_as_uint(big) >> 23, 14u), 254u);
          const float up = __uint_as_float((267u - x) << 23) * sign;
          down = __uint_as_float((x - 13u) << 23);
#pragma unroll
          for (int j = 0; j < CPL / 2; ++j) w[j] = half2_bits(to_f32<XT>(e[2 * j]) * up, to_f32<XT>(e[2 * j + 1]) * up);
        }
        if (row < KP_ROWS) {
          const uint32_t at = smem_u32(q_smem) + ((row >> 7) * KB + (d0 >> 6)) * (128 * 128) + (row & 127) * 128 + ((((d0 & 63) >> 3) ^ (row & 7)) << 4) + (d0 & 7) * 2;
          if constexpr (CPL == 4) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[CPL / 2 - 1]) : "memory");
          else                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w[0]) : "memory");
          if (lane == 0) s_factor[row] = down * fabsf(p.scale);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (idx == rg.begin) PTRACE(2);

    float ref = -INFINITY, m = -INFINITY, l = 0.f;     // of a softmax thread's row: references of O and of l
    if (warp == W_COPY) {
      // ===================== raw codes =====================
      if (lane == 0) {
        bool bad;
        int64_t block = nt > 0 ? block_of(pc.t_first, bad) : 0;
        for (int k = 0; k < nt && ok; ++k) {
          const int tile = pc.t_first + k;
          const int64_t next = k + 1 < nt ? block_of(tile + 1, bad) : 0;      // one ahead
          const int64_t at = ((block << page_shift) + (tile & ((1 << page_shift) - 1))) * (int64_t)UNIT;
          for (int part = 0; part < 2 && ok; ++part) {
            const uint32_t u = 2 * (done + k) + part, slot = u % KP_RAW;
            if (u >= KP_RAW) ok = mbar_wait_suspended(&raw_empty[slot], (u / KP_RAW + 1) & 1, abort_flag);
            if (!ok) break;
            mbar_expect_tx(&raw_full[slot], UNIT);
            bulk_load(smem_u32(raw) + slot * UNIT, (part ? p.v : p.k) + at, UNIT, &raw_full[slot]);
          }
          block = next;
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    } else if (warp == W_MMA) {
      // ===================== MMAs =====================
      const uint32_t idesc_s = make_idesc_f16(0, 0, 0, 128, 64), idesc_o = make_idesc_f16(0, 0, 0, 128, DW);
      const uint64_t dq = make_desc_sw128(smem_u32(q_smem), 16, 1024), dk0 = make_desc_sw128(smem_u32(k_smem), 16, 1024);
      const uint64_t dv0 = make_desc_sw128(smem_u32(v_smem), 16, 1024);
      for (int k = 0; k <= nt && ok; ++k) {
        if (k < nt) {                                  // scores of tile k
          const uint32_t c = done + k, b = c & 1, buf = c % NG;
          ok = __all_sync(0xffffffffu, mbar_wait_suspended(&k_full[buf], (c / NG) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dk = dk0 + (uint32_t)((buf * 64 * DW * 2) >> 4);
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
#pragma unroll
              for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int k16 = 0; k16 < 4; ++k16)
                  mma_f16_ss(tmem + grp * KP_TMEM + 64 * b, dq + (uint32_t)(((grp * KB + kb) * 128 * 128 + k16 * 32) >> 4),
                             dk + (uint32_t)((kb * 64 * 128 + k16 * 32) >> 4), idesc_s, kb > 0 || k16 > 0 ? 1u : 0u);
              if (grp == NG - 1) mma_commit(&k_empty[buf]);
              mma_commit(&s_full[2 * grp + b]);
            }
          }
          __syncwarp();
        }
        if (k > 0) {                                   // outputs of tile k - 1
          const uint32_t c = done + k - 1, b = c & 1, buf = c % NG;
          ok = __all_sync(0xffffffffu, mbar_wait_suspended(&v_full[buf], (c / NG) & 1, abort_flag));
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&p_full[2 * grp + b], (c >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t dv = dv0 + (uint32_t)((buf * 64 * DW * 2) >> 4);
#pragma unroll
              for (int k16 = 0; k16 < 4; ++k16)
                mma_f16_ts(tmem + grp * KP_TMEM + 128, tmem + grp * KP_TMEM + 64 * b + 8 * k16, dv + (uint32_t)((k16 * 32) >> 4), idesc_o,
                           k > 1 || k16 > 0 ? 1u : 0u);
              if (grp == NG - 1) mma_commit(&v_empty[buf]);
              mma_commit(&o_done[2 * grp + b]);
            }
            __syncwarp();
          }
        }
      }
    } else if (warp >= W_EXPAND) {
      // ===================== codes into operands: one or two warps each for keys and values =====================
      const int part = (warp - W_EXPAND) / EW, half = (warp - W_EXPAND) % EW;
      uint64_t *full = part ? v_full : k_full, *empty = part ? v_empty : k_empty;
      // lane's 16-byte piece i = lane + 32 j: row and chunk of the operand; the row's low bits, which swizzle, follow j's parity at most
      constexpr int KP = DW / 16;                      // pieces per row of keys
      const int row0 = part ? lane >> 2 : lane / KP, col = part ? lane & 3 : lane % KP;
      const uint32_t to = smem_u32(part ? v_smem : k_smem) + (part ? 0 : (col >> 2) * (64 * 128)) + row0 * 128;
      const uint32_t row_step = part ? 8 * 128 : (32 / KP) * 128, odd = !part && KP == 8 ? 64u : 0u;
      const uint32_t c0 = ((2 * (col & 3)) ^ (row0 & 7)) << 4, c1 = c0 ^ 16;
      constexpr int STEPS = UNIT / 16 / 32;            // of the operand's warps together
      float vs_next = 1.f;
      if (part && nt > 0) { bool bad; vs_next = p.v_scale[block_of(pc.t_first, bad)]; }
      for (int k = 0; k < nt && ok; ++k) {
        const uint32_t c = done + k, u = 2 * c + part, slot = u % KP_RAW, buf = c % NG;
        const float vs = vs_next;                      // one tile ahead
        if (part && k + 1 < nt) { bool bad; vs_next = p.v_scale[block_of(pc.t_first + k + 1, bad)]; }
        ok = __all_sync(0xffffffffu, mbar_wait_suspended(&raw_full[slot], (u / KP_RAW) & 1, abort_flag));
        if (ok && c >= NG) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&empty[buf], (c / NG + 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t from = smem_u32(raw) + slot * UNIT + lane * 16;
        constexpr int BATCH = STEPS / EW < 8 ? STEPS / EW : 8;      // loads ahead of the stores that they must not pass
        auto expand = [&](auto f) {
#pragma unroll
          for (int j0 = 0; j0 < STEPS / EW; j0 += BATCH) {
            uint4 v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) v[i] = lds16(from + (half * (STEPS / EW) + j0 + i) * 512);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int j = half * (STEPS / EW) + j0 + i;
              const uint32_t at = to + buf * (64 * DW * 2) + j * row_step, x = (j & 1) ? odd : 0u;
              sts16(at + (c0 ^ x), f(v[i].x, 0x4140), f(v[i].x, 0x4342), f(v[i].y, 0x4140), f(v[i].y, 0x4342));
              sts16(at + (c1 ^ x), f(v[i].z, 0x4140), f(v[i].z, 0x4342), f(v[i].w, 0x4140), f(v[i].w, 0x4342));
            }
          }
        };
        if (vs > 0.f) {
          expand([](uint32_t w, uint32_t sel) { return code_pair_f16(w, sel); });
        } else {                                       // values of a zero scale are zero, of a negative one negative
          const uint32_t keep = vs == 0.f ? 0u : 0xffffffffu, flip = vs < 0.f ? 0x80008000u : 0u;
          expand([=](uint32_t w, uint32_t sel) { return (code_pair_f16(w, sel) & keep) ^ flip; });
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) { mbar_arrive(&full[buf]); mbar_arrive(&raw_empty[slot]); }
      }
    } else {
      // ===================== softmax (thread = row) =====================
      const int grp = warp >> 2;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, tmem_s = tmem + grp * KP_TMEM + lanes, tmem_o = tmem_s + 128;
      const float q_factor = s_factor[tid];
      const int limit = tid < pc.rows ? L - n + (p.group == 1 ? pc.c0 + tid : (pc.c0 + tid) / p.group) + 1 : 0;
      const int least = max(0, L - n + (pc.c0 + min(32 * warp, pc.rows - 1)) / p.group + 1);        // what the warp's first row sees
      const bool partial = 32 * warp + 32 > pc.rows;
      bool bad;
      int64_t block = nt > 0 ? block_of(pc.t_first, bad) : 0;
      float ks = nt > 0 ? (bad ? __int_as_float(0x7fc00000) : attend_key_scale(p.k_scale[block])) : 0.f, vs = nt > 0 ? fabsf(p.v_scale[block]) : 0.f, lv = log2f(vs);
      for (int k = 0; k < nt; ++k) {
        const uint32_t c = done + k, b = c & 1;
        const int tile = pc.t_first + k;
        float ks_next = 0.f, vs_next = 0.f;
        if (k + 1 < nt) {
          block = block_of(tile + 1, bad);
          ks_next = bad ? __int_as_float(0x7fc00000) : attend_key_scale(p.k_scale[block]);
          vs_next = fabsf(p.v_scale[block]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&s_full[2 * grp + b], (c >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const bool masked = partial || (tile + 1) * KV_TILE > least;
        const int seen = limit - tile * KV_TILE;       // columns of the tile that this row sees
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t sc[KEEP ? 2 : 1][32];                 // NG = 2: both halves stay in registers
        if (KEEP) {
          tmem_ld_32x32(tmem_s + 64 * b, sc[0]);
          tmem_ld_32x32(tmem_s + 64 * b + 32, sc[KEEP ? 1 : 0]);
          tmem_ld_wait();
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t (&v)[32] = sc[KEEP ? half : 0];
          if (!KEEP) {
            tmem_ld_32x32(tmem_s + 64 * b + 32 * half, v);
            tmem_ld_wait();
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * half + i >= seen) v[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) top4[i & 3] = fmaxf(top4[i & 3], __uint_as_float(v[i]));
        }
        float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        const float f = q_factor * ks;                 // not negative
        top = top == -INFINITY ? top : top * f;
        if (top > m) {
          l *= exp2_fast(m - top);
          m = top;
        }
        const float most = top == -INFINITY || vs == 0.f ? -INFINITY : top + lv;      // values of a zero scale are zero, whatever p' is
        const float now = most > ref + KP_LAZY || ref == -INFINITY ? fmaxf(most, ref) : ref;
        if (__any_sync(0xffffffffu, ref != -INFINITY && now != ref)) {
          // O is complete up to tile k - 1 once that product is done
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&o_done[2 * grp + (b ^ 1)], ((c - 1) >> 1) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const float alpha = ref == -INFINITY ? 1.f : exp2_fast(ref - now);
#pragma unroll
          for (int d = 0; d < DW; d += 32) {
            uint32_t o[32];
            tmem_ld_32x32(tmem_o + d, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32(tmem_o + d, o);
          }
          tmem_st_wait();
        }
        ref = now;
        // p' = 2^(score + lv - ref) = 2^(score - m - back)
        const float back = vs == 0.f || ref == -INFINITY ? 0.f : fminf(ref - lv - m, KP_FAINT), add = (m == -INFINITY ? 0.f : -m - back) + (vs - vs);       // NaN for scales that are not finite
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t (&v)[32] = sc[KEEP ? half : 0];
          uint32_t ph[16];
          if (!KEEP) {
            tmem_ld_32x32(tmem_s + 64 * b + 32 * half, v);
            tmem_ld_wait();
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float a = exp2_fast(fmaf(__uint_as_float(v[2 * i]), f, add)), e = exp2_fast(fmaf(__uint_as_float(v[2 * i + 1]), f, add));
            if (masked) {                              // not even a NaN of the scales reaches a row that does not see the token
              if (32 * half + 2 * i >= seen) a = 0.f;
              if (32 * half + 2 * i + 1 >= seen) e = 0.f;
            }
            sum4[i & 3] += a + e;
            ph[i] = half2_bits(a, e);
          }
          tmem_st_32x16(tmem_s + 64 * b + 16 * half, ph);        // over scores that have been read
        }
        tmem_st_wait();
        const float sum = (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
        if (sum != 0.f) l = fmaf(sum, exp2_fast(back), l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * grp + b]);
        ks = ks_next; vs = vs_next; lv = log2f(vs);
      }

      if (idx == rg.begin) PTRACE(3);
      PTRACE(4);
    }
    done += nt;

    // ---- out: 128 rows at a time by way of shared memory ----
    const bool whole = pc.t_first == 0 && pc.t_last == pc.tiles;
    float* slice = attend_slice<KP_ROWS, DW>(p, rg, blockIdx.x, pc);
    const uint32_t c_last = done - 1;
    if (warp < 4 * NG && ok && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&o_done[2 * (warp >> 2) + (c_last & 1)], (c_last >> 1) & 1, abort_flag));
    if (!ok) l = __int_as_float(0x7fc00000);
    if (warp < 4 * NG) {
      s_ml[tid] = make_float2(m, l);
      s_inv[tid] = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      s_row[tid] = attend_out_row(p, pc, min(tid, pc.rows - 1));
    }
    const float scale_o = exp2_fast(ref - m);
    for (int g0 = 0; g0 < NG && 128 * g0 < pc.rows; ++g0) {
      __syncthreads();                                 // the operands have been read, the rows before have left
      if (warp >> 2 == g0 && warp < 4 * NG) {
        tc_fence_after();
#pragma unroll 1
        for (int d = 0; d < DW; d += 32) {
          uint32_t o[32];
          if (ok && nt > 0) {
            tmem_ld_32x32(tmem + g0 * KP_TMEM + 128 + ((uint32_t)(32 * (warp & 3)) << 16) + d, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          float4* dst = reinterpret_cast<float4*>(staged + (tid & 127) * OST + d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v[4] = {__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])};
            dst[i] = ref == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[0] * scale_o, v[1] * scale_o, v[2] * scale_o, v[3] * scale_o);
          }
        }
        tc_fence_before();
      }
      __syncthreads();
      const int rows = min(128, pc.rows - 128 * g0);
      for (int i = tid; i < rows * (DW / 4); i += KP_THREADS) {
        const int row = i / (DW / 4), d = 4 * (i % (DW / 4)), col = 128 * g0 + row;
        const float4 v = *reinterpret_cast<const float4*>(staged + row * OST + d);
        if (whole) {
          attend_store4<XT>(p, s_row[col], d, v, s_inv[col]);
          if (d == 0 && p.lse) attend_put_lse(p, s_row[col], s_ml[col].x, s_ml[col].y);
        } else {
          *reinterpret_cast<float4*>(slice + col * DW + d) = v;
          if (d == 0) *reinterpret_cast<float2*>(slice + KP_ROWS * DW + 2 * col) = s_ml[col];
        }
      }
    }
    if (!whole) {
      const int first_c = attend_cta_of(pc.tile_at, rg.S, rg.G), last_c = attend_cta_of(pc.tile_at + pc.tiles - 1, rg.S, rg.G);
      if (attend_last(p, first_c, last_c, &s_flag)) attend_join<XT, KP_ROWS, DW, KP_THREADS, NG == 1 ? 3 : 4, 2>(p, rg, pc, first_c, last_c);
    }
    __syncthreads();                                   // before Q and O are written again
    tc_fence_after();
    ok = *abort_flag == 0;
    idx = pc.tile_at + pc.t_last;
  }

  PTRACE(5);
#ifdef JGQ_TRACE
  if (threadIdx.x == 0 && blockIdx.x < 1024) g_trace_prompt[8 * blockIdx.x + 6] = done;
#endif
  // After a wait that ran out copies may still be in flight: a bounded time to land before the shared memory is released.
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000LL) {}
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, NG * KP_TMEM);
  }
}

// ------------------------------------------------------------------ host ----
PromptPlan plan_kv_prompt(int64_t rows, int dw, int q_dtype) {
  PromptPlan pl;
  memset(&pl, 0, sizeof(pl));
  if (rows <= 64 || dw > 128 || q_dtype == JGQ_F32) return pl;
  pl.use = 1;
  pl.groups = rows >= 256 ? 2 : 1;
  pl.G = std::min(KA_TICKETS, (pl.groups == 2 ? 1 : 2) * sm_count());
  pl.slice_bytes = align_up((size_t)pl.G * 2 * 128 * pl.groups * (dw + 2) * sizeof(float), 256);
  return pl;
}

template <typename XT, int DW, int NG>
static int launch_prompt_inst(const PromptPlan& pl, const AttendParams& p, cudaStream_t s) {
  auto kern = kv_prompt_kernel<XT, DW, NG>;
  struct AttrTag {};
  const int arc = once_per_device<AttrTag>([&]() {
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    cudaGetLastError();
    return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kp_smem(DW, NG));
  });
  if (arc != 0) return fail(JGQ_ERR_CUDA, "kv_attend: cannot raise the dynamic shared memory limit");
  kern<<<(unsigned)pl.G, kp_threads(NG), kp_smem(DW, NG), s>>>(p);
  return check_launch("kv_prompt");
}

template <typename XT>
static int launch_prompt(const PromptPlan& pl, const AttendParams& p, int dw, cudaStream_t s) {
  if (dw == 64) return pl.groups == 2 ? launch_prompt_inst<XT, 64, 2>(pl, p, s) : launch_prompt_inst<XT, 64, 1>(pl, p, s);
  return pl.groups == 2 ? launch_prompt_inst<XT, 128, 2>(pl, p, s) : launch_prompt_inst<XT, 128, 1>(pl, p, s);
}

int launch_kv_prompt(const PromptPlan& pl, const AttendParams& p, int dw, int q_dtype, cudaStream_t s) {
  return q_dtype == JGQ_F16 ? launch_prompt<__half>(pl, p, dw, s) : launch_prompt<__nv_bfloat16>(pl, p, dw, s);
}

}  // namespace jgq
