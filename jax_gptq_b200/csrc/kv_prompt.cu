// Attention over the paged 8-bit cache for many rows per sequence (prompts and chunks of them): tcgen05.
//
// An item is 256 rows of q (tokens x heads of one kv head's group) of a sequence and kv head, two groups of 128 (the second may be
// empty), which share the expanded codes; its tiles are 64 tokens.  One CTA per SM.  (With 128 rows per item and two CTAs per SM,
// 160 rows of 64 sequences took 165 us for 132, 100 rows of 4 long ones 84 for 62; 70 rows of 32 shorter ones 69 for 75.)
//   S = Q K^T     M = 128 rows, N = 64 tokens:  Q and the tile's keys in shared memory, S in tensor memory (two buffers)
//   P             softmax warps read S (one row per thread), write p as f16 over it
//   O += P V      M = 128 rows, N = DW channels: P out of tensor memory, the tile's values [channel][token] in shared memory
// The codes become whole numbers (exact) of q's type for the scores, f16 for the values; q stays as it is and comes by TMA (where
// 128 rows are not whole tokens or rows not on 16-byte boundaries, the warps copy it).  Scales meet fp32 numbers: the keys' in
// the scores, the values' in the exponent,
//   p' = 2^(score + log2(v_scale) - reference),
// so that p' is rounded once, and finest where p v_scale is largest, whatever the scales of the pages are.  The row's reference is
// raised only when score + log2(v_scale) passes it by 12 (p' then stays below 2^12), O is rescaled then, by the row's thread; the
// tile's p' are computed with the old reference first and again in that case, so that a tile's scores are read once as a rule.
// The sum of exponentials has a reference of its own, the running maximum of the scores (kept within 2^12): it takes p' before the
// rounding, 64 of them at a time, times 2^(reference - log2(v_scale) - maximum) (two units of 2^-23 off at most, as 2^x is).
//
// Per tile and 128 rows: 512 tensor clocks (DW = 128), 8192 exponentials (512 clocks of the special function unit); a tile of 256 rows takes
// 2650 clocks.  No unit is full (a capture shows the special function unit 26 % busy, the tensor pipe 24 %, issue 43 %): the softmax
// warps' chain bounds it, 1600 clocks between the first score and the last p', in which a thread loads 32 scores, waits for them and
// computes, twice.
// Measured: four chunks of 512 rows, 32 heads of 128, up to 4096 tokens (f16): 95 us, 36 GFLOP; 2048 rows, 16384 tokens, 32 / 8 heads
// (bf16): 645 us, 0.8 PFLOP/s.  Copies of the softmax loop cost more than a second pass over a tile: with three of them 109 and 684 us.
//
// Roles: warps 0 .. 7 softmax, then one warp for copies (q; a ring of four units of raw codes), one that issues the MMAs,
// four (with one 118 us instead of 101) that turn the keys' codes into an operand, two for the values' (128-byte
// swizzle; [token][64 channels] twice, [channel][64 tokens]).  Page numbers are read two tiles ahead, scales one: in front of a tile
// they cost 500 clocks.  All warps write the outputs, by way of shared memory, so that rows go out whole.
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

constexpr int NG = 2;                                  // groups of 128 rows, and buffers of expanded codes
constexpr int KP_THREADS = 512, KP_ROWS = 128 * NG;
constexpr int KP_COST = 5;                             // what an item takes beside its tiles, in tiles (see kv_attend.cu)
constexpr int KP_RAW = 4;                              // raw units (keys or values of a tile) in the ring
constexpr int KP_TMEM = 256;                           // columns per group: S and P 2 x 64, O DW
constexpr float KP_LAZY = 12.f;                        // log2 by which p v_scale may pass its row's reference
constexpr float KP_FAINT = 60.f;                       // log2 below which it is as good as nothing beside the reference

__host__ __device__ constexpr int kp_unit(int dw) { return 64 * dw; }
// q, two buffers of expanded keys and of values, the ring; the outputs take their place at the end of a piece
__host__ __device__ constexpr int kp_operands(int dw) { return KP_ROWS * dw * 2 + 2 * NG * 64 * dw * 2 + KP_RAW * kp_unit(dw); }
__host__ __device__ constexpr int kp_smem(int dw) { return 1024 + 1024 + kp_operands(dw); }

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

// the same as bf16: 128 + the low seven bits, less 256 or, where the top bit is set, 128
__device__ __forceinline__ uint32_t code_pair_bf16(uint32_t w, uint32_t sel) {
  const uint32_t r = __byte_perm(w, 0x43434343u, sel);
  const uint32_t low = r & 0xff7fff7fu, take = (~r & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&take));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename XT, int DW>
__global__ void __launch_bounds__(KP_THREADS, 1)
kv_prompt_kernel(const __grid_constant__ CUtensorMap qmap, const AttendParams p) {
  using namespace umma;
  constexpr int WARPS = KP_THREADS / 32;
  constexpr int UNIT = kp_unit(DW), KB = DW / 64;      // 64-channel blocks of a row
  constexpr int W_COPY = 4 * NG, W_MMA = W_COPY + 1, W_EXPAND = W_COPY + 2;
  constexpr int EWK = 4, EWV = 2;        // warps that expand keys, and values
  static_assert(W_EXPAND + EWK + EWV == WARPS, "every warp has a role");
  constexpr bool BF = std::is_same<XT, __nv_bfloat16>::value;
  constexpr int OST = DW + 4;                          // floats per row of staged outputs
  static_assert(KP_ROWS * OST * 4 <= kp_operands(DW), "the outputs fit the operands' place");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base);
  uint64_t* raw_full = bars, *raw_empty = bars + KP_RAW;
  uint64_t *k_full = bars + 2 * KP_RAW, *k_empty = k_full + NG, *v_full = k_empty + NG, *v_empty = v_full + NG;       // per buffer
  uint64_t *s_full = v_empty + NG, *p_full = s_full + 2 * NG, *o_done = p_full + 2 * NG;         // per group, for even and odd tiles
  uint64_t* q_full = o_done + 2 * NG;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  uint8_t* q_smem = base + 1024;                       // [NG][KB][128 rows][128 bytes], swizzled
  uint8_t* k_smem = q_smem + KP_ROWS * DW * 2;         // [NG buffers][KB][64 tokens][128 bytes]
  uint8_t* v_smem = k_smem + NG * 64 * DW * 2;         // [NG buffers][DW channels][128 bytes]
  uint8_t* raw = v_smem + NG * 64 * DW * 2;
  float* staged = reinterpret_cast<float*>(q_smem);
  __shared__ int64_t s_pre[KP_THREADS + 1];
  __shared__ int64_t s_found[2];
  __shared__ float2 s_ml[KP_ROWS];                     // a row's maximum and sum, when its piece is done,
  __shared__ float s_inv[KP_ROWS];                     // what its outputs are multiplied by,
  __shared__ int64_t s_row[KP_ROWS];                   // and where they go
  __shared__ int s_flag, s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &s_abort;
  PTRACE(0);
  if (tid == 0) {
    for (int i = 0; i < KP_RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], i & 1 ? EWV : EWK); }
    for (int i = 0; i < NG; ++i) { mbar_init(&k_full[i], EWK); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], EWV); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < 2 * NG; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1); }
    mbar_init(q_full, 1);
    s_abort = 0;
    fence_barrier_init();
    if (p.q_map) prefetch_tensormap(&qmap);
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
  uint32_t pieces = 0;                                 // pieces with tiles before this one
  uint32_t done = 0;                                   // tiles of earlier pieces: every role's barriers count on from them
  bool ok = true;

  AttendCursor<KP_ROWS, KP_COST> cursor;
  cursor.find(p, rg);
  for (int64_t idx = rg.begin; idx < rg.end; cursor.next(p, rg)) {
    const AttendPiece pc = cursor.piece(p, rg, idx);
    if (pc.t_last <= pc.t_first) break;                // the item's tiles begin behind this range
    const int n = pc.n, L = pc.L, h = pc.h;
    const int seen_item = max(0, L - n + (pc.c0 + pc.rows - 1) / p.group + 1);
    const int t_end = min(pc.t_last, (seen_item + KV_TILE - 1) / KV_TILE);
    const int nt = max(0, t_end - pc.t_first);         // tiles of this piece
    const bool two = pc.rows > 128;                    // the second group has rows; otherwise its barriers alone go on
    const int32_t* row_of_table = p.table + (int64_t)rg.r * p.table_stride;
    // A tile's scales lie behind its page number: numbers are read two tiles ahead, scales one, so that no warp waits for both.
    auto page_of = [&](int k) { return k < nt ? row_of_table[(pc.t_first + k) >> page_shift] : 0; };
    auto block_of = [&](int page, bool& bad) {         // page and head
      bad = page < 0 || page >= p.pages;
      return (int64_t)(bad ? 0 : page) * p.Hkv + h;
    };

    // ---- q into shared memory: boxes of 64 channels x 128 rows, or where TMA cannot, a warp per row, all of its rows at once ----
    if (!p.q_map) {
      constexpr int CPL = DW / 32, QR = (KP_ROWS + WARPS - 1) / WARPS;         // channels per lane, rows per warp
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
          __align__(8) XT e[CPL];
#pragma unroll
          for (int j = 0; j < CPL; ++j) e[j] = d0 + j < p.D ? src[d0 + j] : from_f32<XT>(0.f);
          raw_q[r] = *reinterpret_cast<const V*>(e);
        }
      }
#pragma unroll
      for (int r = 0; r < QR; ++r) {
        const int row = warp + r * WARPS;
        if (row < KP_ROWS) {
          const uint32_t at = smem_u32(q_smem) + ((row >> 7) * KB + (d0 >> 6)) * (128 * 128) + (row & 127) * 128 + ((((d0 & 63) >> 3) ^ (row & 7)) << 4) + (d0 & 7) * 2;
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw_q[r]);
          if constexpr (CPL == 4) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[CPL / 2 - 1]) : "memory");
          else                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w[0]) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
    }
    if (idx == rg.begin) PTRACE(2);

    float ref = -INFINITY, m = -INFINITY, l = 0.f;     // of a softmax thread's row: references of O and of l
    if (warp == W_COPY) {
      // ===================== raw codes =====================
      if (lane == 0) {
        if (p.q_map && nt > 0) {                       // rows behind the item's are loaded too, and masked
          mbar_expect_tx(q_full, (two ? 2 : 1) * 128 * DW * 2);
          for (int grp = 0; grp < (two ? 2 : 1); ++grp)
            for (int kb = 0; kb < KB; ++kb)
              tma_load_3d(smem_u32(q_smem) + (grp * KB + kb) * (128 * 128), &qmap, 64 * kb, h * p.group, pc.row_first + (pc.c0 + 128 * grp) / p.group, q_full);
        }
        bool bad;
        int page = page_of(0), page_1 = page_of(1);
        for (int k = 0; k < nt && ok; ++k) {
          const int tile = pc.t_first + k, page_2 = page_of(k + 2);
          const int64_t block = block_of(page, bad);
          const int64_t at = ((block << page_shift) + (tile & ((1 << page_shift) - 1))) * (int64_t)UNIT;
          for (int part = 0; part < 2 && ok; ++part) {
            const uint32_t u = 2 * (done + k) + part, slot = u % KP_RAW;
            if (u >= KP_RAW) ok = mbar_wait_suspended(&raw_empty[slot], (u / KP_RAW + 1) & 1, abort_flag);
            if (!ok) break;
            mbar_expect_tx(&raw_full[slot], UNIT);
            bulk_load(smem_u32(raw) + slot * UNIT, (part ? p.v : p.k) + at, UNIT, &raw_full[slot]);
          }
          page = page_1;
          page_1 = page_2;
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    } else if (warp == W_MMA) {
      // ===================== MMAs =====================
      const uint32_t idesc_s = make_idesc_f16(BF ? 1 : 0, 0, 0, 128, 64), idesc_o = make_idesc_f16(0, 0, 0, 128, DW);
      const uint64_t dq = make_desc_sw128(smem_u32(q_smem), 16, 1024), dk0 = make_desc_sw128(smem_u32(k_smem), 16, 1024);
      const uint64_t dv0 = make_desc_sw128(smem_u32(v_smem), 16, 1024);
      if (p.q_map && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait_suspended(q_full, pieces & 1, abort_flag));
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
              if (grp == 0 || two)
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
              if (grp == 0 || two)
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
      // ===================== codes into operands: four warps for the keys', two for the values' =====================
      const int part = warp >= W_EXPAND + EWK, share = part ? warp - W_EXPAND - EWK : warp - W_EXPAND;
      uint64_t *full = part ? v_full : k_full, *empty = part ? v_empty : k_empty;
      // lane's 16-byte piece i = lane + 32 j: row and chunk of the operand; the row's low bits, which swizzle, follow j's parity at most
      constexpr int KP = DW / 16;                      // pieces per row of keys
      const int row0 = part ? lane >> 2 : lane / KP, col = part ? lane & 3 : lane % KP;
      const uint32_t to = smem_u32(part ? v_smem : k_smem) + (part ? 0 : (col >> 2) * (64 * 128)) + row0 * 128;
      const uint32_t row_step = part ? 8 * 128 : (32 / KP) * 128, odd = !part && KP == 8 ? 64u : 0u;
      const uint32_t c0 = ((2 * (col & 3)) ^ (row0 & 7)) << 4, c1 = c0 ^ 16;
      constexpr int STEPS = UNIT / 16 / 32;            // of the operand's warps together
      const float* scales = part ? p.v_scale : p.k_scale;
      float scale_next = 1.f;
      int page_1 = 0;
      bool bad;
      if (nt > 0) { scale_next = scales[block_of(page_of(0), bad)]; page_1 = page_of(1); }
      for (int k = 0; k < nt && ok; ++k) {
        const uint32_t c = done + k, u = 2 * c + part, slot = u % KP_RAW, buf = c % NG;
        const float scale = scale_next;                // one tile ahead
        scale_next = scales[block_of(page_1, bad)];
        page_1 = page_of(k + 2);
        ok = __all_sync(0xffffffffu, mbar_wait_suspended(&raw_full[slot], (u / KP_RAW) & 1, abort_flag));
        if (ok && c >= NG) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&empty[buf], (c / NG + 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t from = smem_u32(raw) + slot * UNIT + lane * 16;
        auto expand = [&](auto ew, auto f) {
          constexpr int MINE = STEPS / decltype(ew)::value, BATCH = MINE < 8 ? MINE : 8;     // loads ahead of the stores that they must not pass
#pragma unroll
          for (int j0 = 0; j0 < MINE; j0 += BATCH) {
            uint4 v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) v[i] = lds16(from + (share * MINE + j0 + i) * 512);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int j = share * MINE + j0 + i;
              const uint32_t at = to + buf * (64 * DW * 2) + j * row_step, x = (MINE % 2 == 0 ? i : j) & 1 ? odd : 0u;
              sts16(at + (c0 ^ x), f(v[i].x, 0x4140), f(v[i].x, 0x4342), f(v[i].y, 0x4140), f(v[i].y, 0x4342));
              sts16(at + (c1 ^ x), f(v[i].z, 0x4140), f(v[i].z, 0x4342), f(v[i].w, 0x4140), f(v[i].w, 0x4342));
            }
          }
        };
        constexpr std::integral_constant<int, EWK> of_k{};
        constexpr std::integral_constant<int, EWV> of_v{};
        auto key = [](uint32_t w, uint32_t sel) { return BF ? code_pair_bf16(w, sel) : code_pair_f16(w, sel); };
        if (!part) {                                   // keys: of q's type, signed as the product of their scale and the scores' is
          if ((p.scale < 0.f) != (scale < 0.f)) expand(of_k, [=](uint32_t w, uint32_t sel) { return key(w, sel) ^ 0x80008000u; });
          else                                  expand(of_k, key);
        } else if (scale > 0.f) {
          expand(of_v, [](uint32_t w, uint32_t sel) { return code_pair_f16(w, sel); });
        } else {                                       // values of a zero scale are zero, of a negative one negative
          const uint32_t keep = scale == 0.f ? 0u : 0xffffffffu, flip = scale < 0.f ? 0x80008000u : 0u;
          expand(of_v, [=](uint32_t w, uint32_t sel) { return (code_pair_f16(w, sel) & keep) ^ flip; });
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) { mbar_arrive(&full[buf]); mbar_arrive(&raw_empty[slot]); }
      }
    } else {
      // ===================== softmax (thread = row) =====================
      const int grp = warp >> 2;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, tmem_s = tmem + grp * KP_TMEM + lanes, tmem_o = tmem_s + 128;
      const float q_factor = fabsf(p.scale);           // positive: a row's maximum is that of its products
      const int limit = tid < pc.rows ? L - n + (p.group == 1 ? pc.c0 + tid : (pc.c0 + tid) / p.group) + 1 : 0;
      const int least = max(0, L - n + (pc.c0 + min(32 * warp, pc.rows - 1)) / p.group + 1);        // what the warp's first row sees
      const bool partial = 32 * warp + 32 > pc.rows;
      bool bad;
      int64_t block = nt > 0 ? block_of(page_of(0), bad) : 0;
      int page_1 = page_of(1);
      float ks = nt > 0 ? (bad ? __int_as_float(0x7fc00000) : attend_key_scale(fabsf(p.k_scale[block]))) : 0.f, vs = nt > 0 ? fabsf(p.v_scale[block]) : 0.f, lv = log2f(vs);
      for (int k = 0; k < nt; ++k) {
        const uint32_t c = done + k, b = c & 1;
        const int tile = pc.t_first + k;
        // the next tile's scales: nothing is done with them before the end of this one
        block = block_of(page_1, bad);
        page_1 = page_of(k + 2);
        const float ks_next = p.k_scale[block], vs_next = p.v_scale[block];
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&s_full[2 * grp + b], (c >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (grp > 0 && !two) {
          if (lane == 0) mbar_arrive(&p_full[2 * grp + b]);
          continue;
        }
        const bool masked = partial || (tile + 1) * KV_TILE > least;
        const int seen = limit - tile * KV_TILE;       // columns of the tile that this row sees
        const float f = q_factor * ks;                 // not negative: the signs are the codes'
        uint32_t ph[32];
        float sum, back;
        // p' = 2^(score + lv - ref) = 2^(score - m - back); a second time where a row needs a new reference (one copy of the code)
#pragma unroll 1
        for (int again = 0;; ++again) {
          back = vs == 0.f || ref == -INFINITY ? 0.f : fminf(ref - lv - m, KP_FAINT);
          const float add = (m == -INFINITY ? 0.f : -m - back) + (vs - vs);       // NaN for scales that are not finite
          float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v[32];
            tmem_ld_32x32(tmem_s + 64 * b + 32 * half, v);
            tmem_ld_wait();
            if (masked) {                              // not even a NaN of the scales reaches a row that does not see the token
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const bool s0 = 32 * half + 2 * i < seen, s1 = 32 * half + 2 * i + 1 < seen;
                const float x = s0 ? __uint_as_float(v[2 * i]) : -INFINITY, y = s1 ? __uint_as_float(v[2 * i + 1]) : -INFINITY;
                const float a = s0 ? exp2_fast(fmaf(x, f, add)) : 0.f, e = s1 ? exp2_fast(fmaf(y, f, add)) : 0.f;
                top4[i & 3] = fmaxf(top4[i & 3], fmaxf(x, y));
                sum4[i & 3] += a + e;
                ph[16 * half + i] = half2_bits(a, e);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float x = __uint_as_float(v[2 * i]), y = __uint_as_float(v[2 * i + 1]);
                const float a = exp2_fast(fmaf(x, f, add)), e = exp2_fast(fmaf(y, f, add));
                top4[i & 3] = fmaxf(top4[i & 3], fmaxf(x, y));
                sum4[i & 3] += a + e;
                ph[16 * half + i] = half2_bits(a, e);
              }
            }
          }
          sum = (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
          if (again) break;
          float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
          top = top == -INFINITY ? top : top * f;
          const float most = top == -INFINITY || vs == 0.f ? -INFINITY : top + lv;      // values of a zero scale are zero, whatever p' is
          const bool up = most > ref + KP_LAZY || (ref == -INFINITY && most > ref), m_up = top > m + KP_LAZY || (m == -INFINITY && top > m);
          if (!__any_sync(0xffffffffu, up || m_up)) break;
          const float now = up ? most : ref;
          if (__any_sync(0xffffffffu, up && ref != -INFINITY)) {
            // O is complete up to tile k - 1 once that product is done
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&o_done[2 * grp + (b ^ 1)], ((c - 1) >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const float alpha = !up || ref == -INFINITY ? 1.f : exp2_fast(ref - now);
#pragma unroll 1
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
          if (m_up) {
            l *= m == -INFINITY ? 1.f : exp2_fast(m - top);
            m = top;
          }
          ref = now;
        }
        if (!ok) break;
#pragma unroll
        for (int half = 0; half < 2; ++half) {         // over scores that have been read
          uint32_t (&w)[16] = *reinterpret_cast<uint32_t (*)[16]>(ph + 16 * half);
          tmem_st_32x16(tmem_s + 64 * b + 16 * half, w);
        }
        tmem_st_wait();
        if (sum != 0.f) l = fmaf(sum, exp2_fast(back), l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * grp + b]);
        ks = bad ? __int_as_float(0x7fc00000) : attend_key_scale(fabsf(ks_next));
        vs = fabsf(vs_next);
        lv = log2f(vs);
      }

      if (idx == rg.begin) PTRACE(3);
      PTRACE(4);
    }
    done += nt;
    pieces += nt > 0;

    // ---- out, by way of shared memory ----
    const bool whole = pc.t_first == 0 && pc.t_last == pc.tiles;
    float* slice = attend_slice<KP_ROWS, DW>(p, rg, blockIdx.x, pc);
    const uint32_t c_last = done - 1;
    // all products are done before anything takes the operands' place
    if (ok && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait_suspended(&o_done[2 * min(warp >> 2, NG - 1) + (c_last & 1)], (c_last >> 1) & 1, abort_flag));
    if (!ok) l = __int_as_float(0x7fc00000);
    __syncthreads();
    if (warp < 4 * NG) {
      s_ml[tid] = make_float2(m, l);
      s_inv[tid] = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      s_row[tid] = attend_out_row(p, pc, min(tid, pc.rows - 1));
      if (128 * (warp >> 2) < pc.rows) {
        const float scale_o = exp2_fast(ref - m);
        tc_fence_after();
#pragma unroll 1
        for (int d = 0; d < DW; d += 32) {
          uint32_t o[32];
          if (ok && nt > 0) {
            tmem_ld_32x32(tmem + (warp >> 2) * KP_TMEM + 128 + ((uint32_t)(32 * (warp & 3)) << 16) + d, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          float4* dst = reinterpret_cast<float4*>(staged + tid * OST + d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v[4] = {__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])};
            dst[i] = ref == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[0] * scale_o, v[1] * scale_o, v[2] * scale_o, v[3] * scale_o);
          }
        }
      }
      tc_fence_before();
    }
    __syncthreads();
    for (int i = tid; i < pc.rows * (DW / 4); i += KP_THREADS) {
      const int row = i / (DW / 4), d = 4 * (i % (DW / 4));
      const float4 v = *reinterpret_cast<const float4*>(staged + row * OST + d);
      if (whole) {
        attend_store4<XT>(p, s_row[row], d, v, s_inv[row]);
        if (d == 0 && p.lse) attend_put_lse(p, s_row[row], s_ml[row].x, s_ml[row].y);
      } else {
        *reinterpret_cast<float4*>(slice + row * DW + d) = v;
        if (d == 0) *reinterpret_cast<float2*>(slice + KP_ROWS * DW + 2 * row) = s_ml[row];
      }
    }
    if (!whole) {
      const int first_c = attend_cta_of(pc.tile_at, rg.S, rg.G), last_c = attend_cta_of(pc.tile_at + pc.tiles - 1, rg.S, rg.G);
      if (attend_last(p, first_c, last_c, &s_flag)) attend_join_rows<XT, KP_ROWS, DW, KP_THREADS, 4, 2>(p, rg, pc, first_c, last_c, s_row, s_ml, s_inv);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the next writers of the staged outputs' place are copies
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
  // 40 rows of 32 sequences, bf16: 67 us here, 63 on mma.sync; of 4 long ones 61 and 66; 64 rows: 71 and 70, 53 and 68; 32 rows: 52 and 52, 46
  // and 44 (kv_attend.cu, with 32 rows per item)
  if (rows <= 32 || dw > 128 || q_dtype == JGQ_F32) return pl;
  pl.use = 1;
  pl.G = std::min(KA_TICKETS, sm_count());
  pl.slice_bytes = align_up((size_t)pl.G * 2 * KP_ROWS * (dw + 2) * sizeof(float), 256);
  return pl;
}

template <typename XT, int DW>
static int launch_prompt_inst(const PromptPlan& pl, const CUtensorMap& qmap, const AttendParams& p, cudaStream_t s) {
  auto kern = kv_prompt_kernel<XT, DW>;
  struct AttrTag {};
  const int arc = once_per_device<AttrTag>([&]() {
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    cudaGetLastError();
    return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kp_smem(DW));
  });
  if (arc != 0) return fail(JGQ_ERR_CUDA, "kv_attend: cannot raise the dynamic shared memory limit");
  kern<<<(unsigned)pl.G, KP_THREADS, kp_smem(DW), s>>>(qmap, p);
  return check_launch("kv_prompt");
}

template <typename XT>
static int launch_prompt(const PromptPlan& pl, const CUtensorMap& qmap, const AttendParams& p, int dw, cudaStream_t s) {
  return dw == 64 ? launch_prompt_inst<XT, 64>(pl, qmap, p, s) : launch_prompt_inst<XT, 128>(pl, qmap, p, s);
}

int launch_kv_prompt(const PromptPlan& pl, AttendParams& p, int dw, int q_dtype, cudaStream_t s) {
  CUtensorMap qmap;
  memset(&qmap, 0, sizeof(qmap));
  // 128 rows of q are whole tokens, and rows lie on 16-byte boundaries; else the warps copy them
  p.q_map = 128 % p.group == 0 && p.vec_q && p.q_token > 0 && p.q_head > 0;
  if (p.q_map) {
    const int rc = encode_tmap_3d_b16(&qmap, p.q, {(uint64_t)p.D, (uint64_t)p.Hq, (uint64_t)p.T}, (uint64_t)p.q_head * 2, (uint64_t)p.q_token * 2, 64,
                                      (uint32_t)p.group, (uint32_t)(128 / p.group));
    if (rc) return rc;
  }
  return q_dtype == JGQ_F16 ? launch_prompt<__half>(pl, qmap, p, dw, s) : launch_prompt<__nv_bfloat16>(pl, qmap, p, dw, s);
}

}  // namespace jgq
