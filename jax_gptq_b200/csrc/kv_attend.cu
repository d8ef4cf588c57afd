// Attention over the paged cache of 8-bit keys and values (layout: kv_cache.cuh).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[t, h] . k_j - max),   j over the tokens that row t may see
//
// Sequence r has lengths[r] tokens in the cache, the last n_r of them are this call's rows (one each, or cu_seqlens[r + 1] -
// cu_seqlens[r]); row i of it sees the first lengths[r] - n_r + i + 1.  A row that sees nothing becomes zeros.
//
// HBM-bound for few rows: every code is read once, 16 bytes per lane, straight into registers, and multiplied by mma.sync with
// the CODES as the 16-row operand and up to 8 NT rows of q (tokens x heads of one kv head's group) as columns.
//   * Operands without conversion: a byte with a zero byte above it is the f16 subnormal byte * 2^-24, which the tensor core
//     multiplies exactly: one byte permute per two codes.  The excess is taken off the sums: 2^24 s - 128 sum(q) for the
//     scores, 2^24 o - 128 sum(p) for the outputs, each once per 64 tokens (sums of 128 |q| lose less than 1e-5 of a score).
//     fp32 calls use exact codes (one f16 subtraction per two codes) and two f16 planes of q and p (22 bits).
//   * The order of the contraction is free as long as both operands agree, so that a lane's 16-byte load is four steps'
//     operands: channels 64 c + 16 t .. + 15 of a key row; tokens 16 t .. + 15 of a value row (stored token-minor).
//   * scores come out as [token][row of q]; the products with the values want [row][token]: two 8 x 8 transposes
//     (movmatrix) per 16 tokens.  The score tiles' token order is chosen so that these are the tokens of a value load.
//   * sum(p) for denominator and excess comes from MMAs with ones, of the very p that the products use (rounded to f16:
//     half a step of 2^-11, as an f16 result is).
//   * running maximum and sum per row (in log2 units), fp32 accumulators; scales meet fp32 numbers only.  p is rounded relative
//     to its tile's maximum, which joins the others in fp32: the weights of a tile keep their precision however faint it
//     is, which counts where its values are larger than others by orders of magnitude.
//
// Keys and values of 64 tokens are contiguous: they come by bulk copies in units of 8 KB (DW = 64: 4 KB), a ring of NSLOT
// units ahead of their use.
//
// Work: the list of all (sequence, kv head, NC rows of q, 64-token tile) is cut into equal contiguous ranges, one per CTA; the
// ranges follow from the lengths on the device.  Two ways to share a CTA's piece of an item among its four warps:
//   few rows (NC = 8 NT): the warps take tiles in turn, each with a ring of its own, and are joined through shared memory;
//   COLS (NC = 32): every warp has eight rows of its own and all walk the same tiles in one ring, refilled by the warp
//   that is the last to have read a unit.  A warp passes over tiles that none of its rows sees.
// An item that several CTAs share is joined by the one that draws the last ticket, in CTA order.  A CTA shares at most two
// items (its first and its last), so two slices per CTA are all the scratch there is.
// Where the rows of a sequence make several row tiles, the earlier ones see fewer tokens: tile counts are a linear function
// rounded down, whose sums have a closed form (floor_sum).
//
// Measured (replayed): 64 sequences up to 32768 tokens, 64 / 8 heads of 128, bf16, one token each (833 MB of codes): 148 us, 5.6 TB/s, 0.86 of
// the measured copy; 700 tokens of one sequence, 12 heads of 64, fp32: 12.5 us, of which the launch and the cut are 3, one tile's chain and
// the join the rest.  Up to 16 rows of 16 bits the warps share tiles (the same bytes for every row), above each has rows of its own.
#include "kv_attend.cuh"
#include "trace.cuh"
#include <algorithm>
#include <cstring>
#include <type_traits>

// measurement builds, per CTA: 0 entry, 1 range known, 2 first piece's tiles done, 3 first piece done, 4 last piece's tiles done, 5 exit
JGQ_TRACE_DEFINE(attend, 8 * 1024)
#define ATRACE(i) JGQ_TRACE_CTA(attend, i, 1024)

namespace jgq {

constexpr int KA_WARPS = 4, KA_THREADS = 32 * KA_WARPS;

// two codes of a word as f16: as subnormals with their excess, or exact
template <bool EXACT>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int upper) {
  if (!EXACT) return __byte_perm(w, 0u, upper ? 0x4342 : 0x4140);
  uint32_t r = __byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140);         // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__float2half_rn(1152.f)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__host__ __device__ constexpr int attend_unit(int dw) { return dw == 64 ? 4096 : 8192; }      // bytes
__host__ __device__ constexpr int attend_slots(int dw, bool cols) { return cols ? (dw == 64 ? 8 : 6) : (dw == 64 ? 4 : dw == 128 ? 2 : 3); }   // units per ring
__host__ __device__ constexpr int attend_ctas(int dw, int nt, bool f32, bool cols) { return cols ? (dw == 64 && nt == 1 ? 3 : 2) : (dw <= 128 && nt == 1 && !f32 ? 3 : 2); }
__host__ __device__ constexpr int attend_ring_bytes(int dw, bool cols) { return attend_unit(dw) * attend_slots(dw, cols) * (cols ? 1 : KA_WARPS); }
__host__ __device__ constexpr int attend_smem(int dw, bool cols) {
  return 1024 + attend_ring_bytes(dw, cols);
}

template <typename XT, int DW, int NT, bool COLS>
__global__ void __launch_bounds__(KA_THREADS, attend_ctas(DW, NT, std::is_same<XT, float>::value, COLS))
kv_attend_kernel(const AttendParams p) {
  using namespace umma;
  constexpr bool F32 = std::is_same<XT, float>::value;
  constexpr bool EXACT = F32;
  constexpr int QP = F32 ? 2 : 1;                      // planes of q and of p
  // What beginning and finishing an item takes, in tiles: units in front of its tiles that only weigh in the cut.  Without
  // them a CTA with many short sequences took 215 us where the others took 119.
  constexpr int kPieceCost = COLS ? 8 : 6;
  constexpr int NC = 8 * NT * (COLS ? KA_WARPS : 1);   // rows of q per item
  constexpr int CH = DW / 64;                          // 64-channel chunks of a row
  constexpr int DT = DW / 16;                          // 16-channel tiles of the output
  constexpr int UNIT = attend_unit(DW), NSLOT = attend_slots(DW, COLS);
  constexpr int UPT = 2 * 64 * DW / UNIT, KU = UPT / 2;                // units per tile; of keys
  constexpr int DTU = DT / KU;                         // channel tiles per unit of values
  constexpr float UP24 = EXACT ? 1.f : 16777216.f;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint64_t* full_all = reinterpret_cast<uint64_t*>(smem_raw);          // [rings][NSLOT]
  int* done = reinterpret_cast<int*>(smem_raw + 512);                  // [NSLOT] warps that have read a unit (COLS)
  uint8_t* ring_all = smem_raw + 1024;
  // few rows: a warp's sums [NC][DW] lie in its own ring, which is empty by then
  static_assert(COLS || NC * DW * 4 <= NSLOT * UNIT, "a warp's sums fit its ring");
  auto sums_of = [&](int w) { return reinterpret_cast<float*>(ring_all + w * (NSLOT * UNIT)); };
  __shared__ __align__(16) float sml[COLS ? 1 : KA_WARPS * NC * 2];                  // [warp][NC] maximum, sum
  __shared__ int64_t s_pre[KA_THREADS + 1];
  __shared__ int64_t s_found[2];
  __shared__ int s_flag, s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  volatile int* abort_flag = &s_abort;
  ATRACE(0);
  if (tid == 0) {
    for (int i = 0; i < NSLOT * (COLS ? 1 : KA_WARPS); ++i) mbar_init(&full_all[i], 1);
    for (int i = 0; i < NSLOT; ++i) done[i] = 0;
    s_abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  attend_zero_rest<XT, KA_THREADS>(p);
  AttendRange rg = attend_range<NC, kPieceCost, KA_THREADS>(p, kPieceCost + KA_WARPS, s_pre, s_found);
  if ((int)blockIdx.x >= rg.G) return;
  uint64_t* full = full_all + (COLS ? 0 : warp * NSLOT);
  const uint32_t ring = smem_u32(ring_all) + (COLS ? 0 : warp * NSLOT * UNIT);
  int slot = 0;                                        // of the ring's next unit, and the parity its arrival has
  uint32_t phase = 0;
  bool alive = true;
  ATRACE(1);
  const int page_shift = p.P == 64 ? 0 : p.P == 128 ? 1 : 2;          // tiles per page

  // ---- pieces: the part of one item (sequence, head, row tile) in this range ----
  AttendCursor<NC, kPieceCost> cursor;
  cursor.find(p, rg);
  for (int64_t idx = rg.begin; idx < rg.end; cursor.next(p, rg)) {
    const AttendPiece pc = cursor.piece(p, rg, idx);
    if (pc.t_last <= pc.t_first) break;                // the item's tiles begin behind this range
    const int n = pc.n, L = pc.L, h = pc.h, c0 = pc.c0, rows = pc.rows, row_first = pc.row_first, t_first = pc.t_first, t_last = pc.t_last;
    const int w0 = COLS ? 8 * NT * warp : 0;           // this warp's first one
    const int mine = COLS ? max(0, min(8 * NT, rows - w0)) : rows;
    // tokens that the first and the last of this warp's rows see, and the last of the item's
    const int seen_least = max(0, L - n + (c0 + w0) / p.group + 1);
    const int seen_most = mine > 0 ? max(0, L - n + (c0 + w0 + mine - 1) / p.group + 1) : 0;
    const int seen_item = max(0, L - n + (c0 + rows - 1) / p.group + 1);
    const int t_end = min(t_last, (seen_item + KV_TILE - 1) / KV_TILE);

    // ---- the ring: unit i of this piece's tiles ----
    const int t_begin = COLS ? t_first : t_first + warp, t_step = COLS ? 1 : KA_WARPS;
    const int my_tiles = t_begin < t_end ? (t_end - t_begin + t_step - 1) / t_step : 0;
    const int32_t* row_of_table = p.table + (int64_t)rg.r * p.table_stride;
    auto page_of = [&](int k) { return k < my_tiles ? row_of_table[(t_begin + k * t_step) >> page_shift] : -1; };
    auto issue = [&](int to, int k, int part, int page) {         // part `part` of tile k, on that page, into a slot; one lane
      const int tile = t_begin + k * t_step;
      const int64_t block = (int64_t)(page < 0 || page >= p.pages ? 0 : page) * p.Hkv + h;
      const int64_t at = ((block << page_shift) + (tile & ((1 << page_shift) - 1))) * (int64_t)(DW * KV_TILE) + (part % KU) * UNIT;
      mbar_expect_tx(&full[to], UNIT);
      bulk_load(ring + to * UNIT, (part < KU ? p.k : p.v) + at, UNIT, &full[to]);
    };
    int page_now = page_of(0), page_1 = page_of(1), page_2 = page_of(2);
    // Tiles in front of the ring's end: units are requested NSLOT ahead, that is up to AHEAD tiles.
    constexpr int AHEAD = (NSLOT + UPT - 1) / UPT;
    static_assert(AHEAD <= 4, "page numbers are kept two tiles ahead, further ones are looked up");
    if (alive && lane == 0 && (!COLS || warp == 0)) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
#pragma unroll
      for (int i = 0; i < NSLOT; ++i)
        if (i / UPT < my_tiles)
          issue(slot + i < NSLOT ? slot + i : slot + i - NSLOT, i / UPT, i % UPT, i / UPT == 0 ? page_now : i / UPT == 1 ? page_1 : i / UPT == 2 ? page_2 : page_of(i / UPT));
    }

    // ---- q: the lane's operands, and per column (2 t, 2 t + 1 of each octet) limit, factor and sum ----
    uint32_t qf[NT][QP][CH][4][2];
    int limit[NT][2];
    float qscale[NT][2], qbias[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[CH][16], big = 0.f, sum = 0.f;
      const int c = 8 * nt + g, row = c0 + w0 + c;
      const bool live = c < mine;
      const XT* src = reinterpret_cast<const XT*>(p.q) + (int64_t)(row_first + (live ? row / p.group : 0)) * p.q_token +
                      (int64_t)(h * p.group + (live ? row % p.group : 0)) * p.q_head;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int d = 64 * ch + 16 * t;
        if (live && p.vec_q && d + 16 <= p.D) {
          __align__(16) XT e[16];
#pragma unroll
          for (int v = 0; v < (int)sizeof(XT); ++v) reinterpret_cast<uint4*>(e)[v] = reinterpret_cast<const uint4*>(src + d)[v];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[ch][i] = to_f32<XT>(e[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[ch][i] = (live && d + i < p.D) ? to_f32<XT>(src[d + i]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(x[ch][i]));
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // a power of two brings the row's largest element to [2^13, 2^14): f16 then holds what bf16 or 22 bits of fp32 say
      const uint32_t e = min(max(__float_as_uint(big) >> 23, 14u), 254u);
      const float up = __uint_as_float((267u - e) << 23), down = __uint_as_float((e - 13u) << 23);
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float x0 = x[ch][4 * j + 2 * b] * up, x1 = x[ch][4 * j + 2 * b + 1] * up;
            const uint32_t hi = half2_bits(x0, x1);
            const float2 f = half2_floats(hi);
            qf[nt][0][ch][j][b] = hi;
            sum += f.x + f.y;
            if (QP == 2) qf[nt][QP - 1][ch][j][b] = half2_bits(x0 - f.x, x1 - f.y);
          }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float f = down * p.scale;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int from = (2 * t + b) * 4, col = 8 * nt + 2 * t + b;
        const float fc = __shfl_sync(0xffffffffu, f, from);
        qscale[nt][b] = fc * UP24;
        qbias[nt][b] = EXACT ? 0.f : -128.f * __shfl_sync(0xffffffffu, sum, from) * fc;
        limit[nt][b] = col < mine ? L - n + (c0 + w0 + col) / p.group + 1 : 0;
      }
    }

    float o[DT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nt][e] = 0.f;
    }

    // ---- tiles ----
    // `ahead` units behind the ring's next one: its slot and parity
    auto slot_of = [&](int ahead) { return slot + ahead < NSLOT ? slot + ahead : slot + ahead - NSLOT; };
    auto wait_unit = [&](int ahead) {
      const uint32_t ph = slot + ahead < NSLOT ? phase : phase ^ 1u;
      if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&full[slot_of(ahead)], ph, abort_flag));
      return ring + (uint32_t)slot_of(ahead) * UNIT;
    };
    // gives back the ring's next unit, part `part` of tile k, and has the one NSLOT further on fetched into its place
    auto pass_unit = [&](int k, int part) {
      __syncwarp();
      if (lane == 0 && alive) {
        bool refill = true;
        if (COLS) {
          int old;
          asm volatile("atom.acq_rel.cta.shared.add.u32 %0, [%1], 1;" : "=r"(old) : "r"(smem_u32(&done[slot])) : "memory");
          refill = old == KA_WARPS - 1;                // every warp has read the unit
          if (refill) done[slot] = 0;
        }
        const int ahead = part + NSLOT, k2 = k + ahead / UPT;
        if (refill && k2 < my_tiles) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          issue(slot, k2, ahead % UPT, ahead / UPT == 0 ? page_now : ahead / UPT == 1 ? page_1 : ahead / UPT == 2 ? page_2 : page_of(k2));
        }
      }
      if (++slot == NSLOT) { slot = 0; phase ^= 1u; }
    };
    const uint32_t k_lane = (uint32_t)((16 * (g >> 1) + (g & 1)) * DW + 16 * t), v_lane = (uint32_t)(64 * g + 16 * t);
    float ks = 0.f, vs = 0.f;
    if (my_tiles > 0) {
      const bool bad = page_now < 0 || page_now >= p.pages;            // no such page: the result is NaN
      const int64_t block = (int64_t)(bad ? 0 : page_now) * p.Hkv + h;
      ks = bad ? __int_as_float(0x7fc00000) : attend_key_scale(p.k_scale[block]);
      vs = p.v_scale[block];
    }
    for (int k = 0; k < my_tiles; ++k) {
      const int tile = t_begin + k * t_step;
      // scales of the next tile, page number of the one after the next
      float ks_next = 0.f, vs_next = 0.f;
      const int page_3 = page_of(k + 3);
      if (k + 1 < my_tiles) {
        const bool bad = page_1 < 0 || page_1 >= p.pages;
        const int64_t block = (int64_t)(bad ? 0 : page_1) * p.Hkv + h;
        ks_next = bad ? __int_as_float(0x7fc00000) : attend_key_scale(p.k_scale[block]);
        vs_next = p.v_scale[block];
      }
      if (COLS && tile * KV_TILE >= seen_most) {       // nothing for this warp's rows
#pragma unroll
        for (int part = 0; part < UPT; ++part) { wait_unit(0); pass_unit(k, part); }
      } else {
        // scores of 64 tokens: tile i has tokens 16 (g / 2) + 4 i + (g & 1), and those plus two
        float s[4][NT][4];
#pragma unroll
        for (int part = 0; part < KU; ++part) wait_unit(part);
        if (alive) {
          const uint32_t slot0 = ring + (uint32_t)slot * UNIT, slot1 = ring + (uint32_t)slot_of(KU - 1) * UNIT;
          // rows 16 (g / 2) + ..: with two units of 32 tokens, lanes g < 4 read the first and g >= 4 the second
          const uint32_t at = KU == 1 ? slot0 + k_lane : (g < 4 ? slot0 + k_lane : slot1 + k_lane - 32 * DW);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
              const uint4 wa = lds16(at + 4 * i * DW + 64 * ch), wb = lds16(at + (4 * i + 2) * DW + 64 * ch);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t a0 = code_pair<EXACT>(word_of(wa, j), 0), a2 = code_pair<EXACT>(word_of(wa, j), 1);
                const uint32_t a1 = code_pair<EXACT>(word_of(wb, j), 0), a3 = code_pair<EXACT>(word_of(wb, j), 1);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int pl = 0; pl < QP; ++pl) {
                    if (ch == 0 && j == 0 && pl == 0) mma_h0(s[i][nt], a0, a1, a2, a3, qf[nt][pl][ch][j][0], qf[nt][pl][ch][j][1]);
                    else                              mma_h(s[i][nt], a0, a1, a2, a3, qf[nt][pl][ch][j][0], qf[nt][pl][ch][j][1]);
                  }
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[i][nt][e] = __int_as_float(0x7fc00000);
        }
#pragma unroll
        for (int part = 0; part < KU; ++part) pass_unit(k, part);
        const bool masked = (tile + 1) * KV_TILE > seen_least;
        uint32_t pb[4][NT][QP][2];                       // p as operands of the products with the values
        float alpha[NT][2], psum[NT][2], vsc[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float top[2] = {-INFINITY, -INFINITY}, down[2];
          const float fs[2] = {qscale[nt][0] * ks, qscale[nt][1] * ks}, fb[2] = {qbias[nt][0] * ks, qbias[nt][1] * ks};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = fmaf(s[i][nt][e], fs[e & 1], fb[e & 1]);
              if (masked && tile * KV_TILE + 16 * (g >> 1) + 4 * i + (g & 1) + (e & 2) >= limit[nt][e & 1]) v = -INFINITY;
              s[i][nt][e] = v;
              top[e & 1] = fmaxf(top[e & 1], v);         // passes a NaN over: its p is one
            }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top[b] = fmaxf(top[b], __shfl_xor_sync(0xffffffffu, top[b], x));
            const float now = fmaxf(m[nt][b], top[b]), ref = now == -INFINITY ? 0.f : now;
            alpha[nt][b] = exp2_fast(m[nt][b] - ref);
            down[b] = exp2_fast(top[b] - ref);
            m[nt][b] = now;
            if (top[b] == -INFINITY) top[b] = 0.f;
          }
          float ones[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float pv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pv[e] = exp2_fast(s[i][nt][e] - top[e & 1]);
            uint32_t ra = half2_bits(pv[0], pv[1]), rb = half2_bits(pv[2], pv[3]);
            pb[i][nt][0][0] = transpose8x8(ra);
            pb[i][nt][0][1] = transpose8x8(rb);
            mma_h(ones, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, pb[i][nt][0][0], pb[i][nt][0][1]);
            if (QP == 2) {
              const float2 fa = half2_floats(ra), fb = half2_floats(rb);
              pb[i][nt][QP - 1][0] = transpose8x8(half2_bits(pv[0] - fa.x, pv[1] - fa.y));
              pb[i][nt][QP - 1][1] = transpose8x8(half2_bits(pv[2] - fb.x, pv[3] - fb.y));
              mma_h(ones, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, pb[i][nt][QP - 1][0], pb[i][nt][QP - 1][1]);
            }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            l[nt][b] = fmaf(l[nt][b], alpha[nt][b], ones[b] * down[b]);
            psum[nt][b] = EXACT ? 0.f : -128.f * ones[b];
            vsc[nt][b] = ones[b] == 0.f ? 0.f : vs * down[b];      // a row that sees none of the tile takes nothing of it, not even a NaN
          }
        }
        bool same = true;                              // no row's maximum grew: the sums stay as they are
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) same &= alpha[nt][0] == 1.f && alpha[nt][1] == 1.f;
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][nt][e] *= alpha[nt][e & 1];
        }
#pragma unroll
        for (int part = 0; part < KU; ++part) {
          const uint32_t at = wait_unit(0) + v_lane;
#pragma unroll
          for (int ii = 0; ii < DTU; ++ii) {
            const int d = part * DTU + ii;
            const uint4 wa = lds16(at + ii * 1024), wb = lds16(at + ii * 1024 + 512);
            float x[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = code_pair<EXACT>(word_of(wa, i), 0), a2 = code_pair<EXACT>(word_of(wa, i), 1);
              const uint32_t a1 = code_pair<EXACT>(word_of(wb, i), 0), a3 = code_pair<EXACT>(word_of(wb, i), 1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int pl = 0; pl < QP; ++pl) {
                  if (i == 0 && pl == 0) mma_h0(x[nt], a0, a1, a2, a3, pb[i][nt][pl][0], pb[i][nt][pl][1]);
                  else                   mma_h(x[nt], a0, a1, a2, a3, pb[i][nt][pl][0], pb[i][nt][pl][1]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[d][nt][e] = fmaf(fmaf(x[nt][e], UP24, psum[nt][e & 1]), vsc[nt][e & 1], o[d][nt][e]);
          }
          pass_unit(k, KU + part);
        }
      }
      page_now = page_1; page_1 = page_2; page_2 = page_3;
      ks = ks_next; vs = vs_next;
    }
    if (idx == rg.begin) ATRACE(2);
    ATRACE(4);
    if (!alive) {                                      // a wait ran out: the result says so
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7fc00000);
    }

    // ---- out ----
    const bool whole = t_first == 0 && t_last == pc.tiles;
    float* slice = attend_slice<NC, DW>(p, rg, blockIdx.x, pc);
    if (COLS) {
      // every warp has all of its rows' tokens here
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (whole) {
          float f[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int c = 8 * nt + 2 * t + b;
            f[b] = l[nt][b] == 0.f ? 0.f : __fdiv_rn(1.f, l[nt][b]);
            if (g == 0 && c < mine && p.lse) attend_put_lse(p, attend_out_row(p, pc, w0 + c), m[nt][b], l[nt][b]);
          }
          if (F32) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int c = 8 * nt + 2 * t + b;
              if (c < mine) {
                XT* dst = reinterpret_cast<XT*>(p.out) + attend_out_row(p, pc, w0 + c) * p.D;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (16 * d + 8 * e + g < p.D) dst[16 * d + 8 * e + g] = from_f32<XT>(o[d][nt][2 * e + b] * f[b]);
              }
            }
          } else {
            // transposed eight by eight: two neighbouring channels of row g per lane
            const int c = 8 * nt + g;
            XT* dst = reinterpret_cast<XT*>(p.out) + (c < mine ? attend_out_row(p, pc, w0 + c) * p.D : 0);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const XT pr[2] = {from_f32<XT>(o[d][nt][2 * e] * f[0]), from_f32<XT>(o[d][nt][2 * e + 1] * f[1])};
                const uint32_t w = transpose8x8((uint32_t)*reinterpret_cast<const uint16_t*>(&pr[0]) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&pr[1]) << 16));
                const int ch = 16 * d + 8 * e + 2 * t;
                if (c < mine && ch < p.D) {
                  if (p.vec_o) *reinterpret_cast<uint32_t*>(dst + ch) = w;
                  else {
                    reinterpret_cast<uint16_t*>(dst)[ch] = (uint16_t)w;
                    if (ch + 1 < p.D) reinterpret_cast<uint16_t*>(dst)[ch + 1] = (uint16_t)(w >> 16);
                  }
                }
              }
          }
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int c = 8 * nt + 2 * t + b, col = w0 + c;
            if (c < mine) {
#pragma unroll
              for (int d = 0; d < DT; ++d) {
                slice[col * DW + 16 * d + g] = o[d][nt][b];
                slice[col * DW + 16 * d + 8 + g] = o[d][nt][2 + b];
              }
              if (g == 0) { slice[NC * DW + 2 * col] = m[nt][b]; slice[NC * DW + 2 * col + 1] = l[nt][b]; }
            }
          }
        }
      }
    } else {
      // join the warps: columns' sums through shared memory
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int col = 8 * nt + 2 * t + b;
          float* dst = sums_of(warp) + col * DW;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            dst[16 * d + g] = o[d][nt][b];
            dst[16 * d + 8 + g] = o[d][nt][2 + b];
          }
          if (g == 0) { sml[(warp * NC + col) * 2] = m[nt][b]; sml[(warp * NC + col) * 2 + 1] = l[nt][b]; }
        }
      __syncthreads();
      for (int i = tid; i < rows * (DW / 4); i += KA_THREADS) {
        const int col = i / (DW / 4), d = 4 * (i % (DW / 4));
        float2 ml[KA_WARPS];
        float mx = -INFINITY, den = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KA_WARPS; ++w) { ml[w] = *reinterpret_cast<const float2*>(&sml[(w * NC + col) * 2]); mx = fmaxf(mx, ml[w].x); }
        const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int w = 0; w < KA_WARPS; ++w) {
          const float f = exp2_fast(ml[w].x - ref);
          const float4 v = *reinterpret_cast<const float4*>(sums_of(w) + col * DW + d);
          sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y); sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
          den = fmaf(ml[w].y, f, den);
        }
        if (whole) {
          attend_finish4<XT>(p, pc, col, d, sum, mx, den);
        } else {
          *reinterpret_cast<float4*>(slice + col * DW + d) = sum;
          if (d == 0) *reinterpret_cast<float2*>(slice + NC * DW + 2 * col) = make_float2(mx, den);
        }
      }
    }
    if (!whole) {
      const int first_c = attend_cta_of(pc.tile_at, rg.S, rg.G), last_c = attend_cta_of(pc.tile_at + pc.tiles - 1, rg.S, rg.G);
      if (attend_last(p, first_c, last_c, &s_flag)) attend_join<XT, NC, DW, KA_THREADS, COLS ? 8 : (NC * DW / 4 + KA_THREADS - 1) / KA_THREADS, COLS ? 2 : 4>(p, rg, pc, first_c, last_c);
    }
    if (idx == rg.begin) ATRACE(3);
    __syncthreads();                                   // before the rings are filled again
    idx = pc.tile_at + t_last;
  }

  ATRACE(5);
  // After a wait that ran out copies may still be in flight: a bounded time to land before the shared memory is released.
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000LL) {}
  }
}

// ------------------------------------------------------------------ host ----
struct AttendPlan { int nt, cols, G; size_t slice_bytes; PromptPlan prompt; };

static AttendPlan plan_attend(int64_t max_new, int64_t group, int dw, int x_dtype) {
  AttendPlan pl;
  const int64_t rows = max_new * group;
  const bool one = dw == 256 || x_dtype == JGQ_F32;    // more accumulators than eight rows' do not fit the registers
  pl.cols = rows > (one ? 8 : 16);
  pl.nt = !one && rows > 8 && !pl.cols ? 2 : 1;
  const int nc = 8 * pl.nt * (pl.cols ? KA_WARPS : 1);
  pl.G = std::min(KA_TICKETS, attend_ctas(dw, pl.nt, x_dtype == JGQ_F32, pl.cols != 0) * sm_count());
  pl.slice_bytes = align_up((size_t)pl.G * 2 * nc * (dw + 2) * sizeof(float), 256);
  pl.prompt = plan_kv_prompt(rows, dw, x_dtype);
  if (pl.prompt.use) pl.slice_bytes = pl.prompt.slice_bytes;
  return pl;
}

template <typename XT, int DW, int NT, bool COLS>
static int launch_attend_inst(const AttendPlan& pl, const AttendParams& p, cudaStream_t s) {
  auto kern = kv_attend_kernel<XT, DW, NT, COLS>;
  constexpr int smem = attend_smem(DW, COLS);
  struct AttrTag {};
  const int arc = once_per_device<AttrTag>([&]() {
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    cudaGetLastError();
    return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (arc != 0) return fail(JGQ_ERR_CUDA, "kv_attend: cannot raise the dynamic shared memory limit");
  kern<<<(unsigned)pl.G, KA_THREADS, smem, s>>>(p);
  return check_launch("kv_attend");
}

template <typename XT, int DW>
static int launch_attend_width(const AttendPlan& pl, const AttendParams& p, cudaStream_t s) {
  if constexpr (!std::is_same<XT, float>::value && DW <= 128) {
    if (pl.nt == 2) return launch_attend_inst<XT, DW, 2, false>(pl, p, s);
  }
  return pl.cols ? launch_attend_inst<XT, DW, 1, true>(pl, p, s) : launch_attend_inst<XT, DW, 1, false>(pl, p, s);
}

template <typename XT>
static int launch_attend(const AttendPlan& pl, const AttendParams& p, int dw, cudaStream_t s) {
  if (dw == 64) return launch_attend_width<XT, 64>(pl, p, s);
  if (dw == 128) return launch_attend_width<XT, 128>(pl, p, s);
  return launch_attend_width<XT, 256>(pl, p, s);
}

}  // namespace jgq

using namespace jgq;

extern "C" size_t jgq_kv_attend_workspace_bytes(int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_new, int q_dtype) {
  if (q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_new <= 0 || q_heads % kv_heads != 0) return 0;
  const AttendPlan pl = plan_attend(max_new, q_heads / kv_heads, kv_width(head_dim), q_dtype);
  return KA_TICKETS * sizeof(int32_t) + pl.slice_bytes;
}

extern "C" int jgq_kv_attend(const void* q, int q_dtype, int64_t q_token_stride, int64_t q_head_stride, void* out, float* lse,
                             const uint8_t* k, const uint8_t* v, const float* k_scale, const float* v_scale, int64_t pages, int page_size,
                             const int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* lengths,
                             const int32_t* cu_seqlens, int64_t tokens, int64_t requests, int64_t max_new,
                             int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scale, int flags,
                             void* ws, size_t ws_bytes, void* stream) {
  JGQ_REQUIRE((flags & ~JGQ_KV_ZERO_REST) == 0, JGQ_ERR_ARG, "kv_attend: unknown flag bits %d", flags);
  JGQ_REQUIRE(q_dtype == JGQ_F32 || q_dtype == JGQ_F16 || q_dtype == JGQ_BF16, JGQ_ERR_ARG, "kv_attend: q dtype must be f32/f16/bf16");
  JGQ_REQUIRE(kv_page_ok(page_size), JGQ_ERR_ARG, "kv_attend: page_size %d is not 64, 128 or 256", page_size);
  JGQ_REQUIRE(head_dim >= 1 && head_dim <= 256, JGQ_ERR_ARG, "kv_attend: head_dim %lld not in [1, 256]", (long long)head_dim);
  JGQ_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0, JGQ_ERR_ARG, "kv_attend: %lld query heads are no multiple of %lld kv heads",
              (long long)q_heads, (long long)kv_heads);
  JGQ_REQUIRE(tokens >= 0 && requests >= 0 && pages > 0 && table_width >= 0 && max_new >= 1, JGQ_ERR_ARG, "kv_attend: bad sizes");
  JGQ_REQUIRE(cu_seqlens || tokens == requests, JGQ_ERR_ARG, "kv_attend: %lld tokens for %lld requests without cu_seqlens", (long long)tokens, (long long)requests);
  JGQ_REQUIRE(tokens <= (1 << 24) && requests <= (1 << 20) && q_heads <= 4096 && tokens * (q_heads / kv_heads) <= 2147483647LL - 1024 &&
                  pages <= 2147483647LL && table_width * page_size <= 2147483647LL - 64,
              JGQ_ERR_LIMIT, "kv_attend: shape too large");
  if (tokens == 0) return JGQ_OK;
  JGQ_REQUIRE(q && out && k && v && k_scale && v_scale && (requests == 0 || (lengths && (block_table || table_width == 0))), JGQ_ERR_ARG, "kv_attend: null pointer");
  const size_t xb = dtype_size(q_dtype);
  JGQ_REQUIRE(aligned(q, xb) && aligned(out, xb) && aligned(k, 16) && aligned(v, 16), JGQ_ERR_ALIGN, "kv_attend: misaligned pointer");
  const size_t need = jgq_kv_attend_workspace_bytes(q_heads, kv_heads, head_dim, max_new, q_dtype);
  JGQ_REQUIRE(ws && ws_bytes >= need, JGQ_ERR_WORKSPACE, "kv_attend: workspace %zu < %zu bytes", ws_bytes, need);
  JGQ_REQUIRE(aligned(ws, 256), JGQ_ERR_ALIGN, "kv_attend: workspace must be 256-byte aligned");
  const int dw = kv_width(head_dim);
  const AttendPlan pl = plan_attend(max_new, q_heads / kv_heads, dw, q_dtype);
  AttendParams p;
  memset(&p, 0, sizeof(p));
  p.q = q; p.out = out; p.lse = lse; p.k = k; p.v = v; p.k_scale = k_scale; p.v_scale = v_scale;
  p.table = block_table; p.lengths = lengths; p.cu = cu_seqlens;
  p.q_token = q_token_stride; p.q_head = q_head_stride; p.table_stride = table_stride;
  p.tickets = (int32_t*)ws; p.slices = (float*)((char*)ws + KA_TICKETS * sizeof(int32_t));
  p.T = (int)tokens; p.B = (int)requests; p.W = (int)table_width; p.Hq = (int)q_heads; p.Hkv = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads); p.D = (int)head_dim; p.P = page_size; p.pages = (int)pages;
  p.vec_q = aligned(q, 16) && q_token_stride * xb % 16 == 0 && q_head_stride * xb % 16 == 0;
  p.vec_o = head_dim % 4 == 0 && aligned(out, 4 * xb);
  p.zero_rest = (flags & JGQ_KV_ZERO_REST) != 0;
  p.G = pl.prompt.use ? pl.prompt.G : pl.G;
  p.scale = scale * 1.4426950408889634f;
  cudaStream_t s = (cudaStream_t)stream;
  if (pl.prompt.use) return launch_kv_prompt(pl.prompt, p, dw, q_dtype, s);
  if (q_dtype == JGQ_F32) return launch_attend<float>(pl, p, dw, s);
  if (q_dtype == JGQ_F16) return launch_attend<__half>(pl, p, dw, s);
  return launch_attend<__nv_bfloat16>(pl, p, dw, s);
}
