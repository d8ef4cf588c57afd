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
//   * running maximum and sum per row (in log2 units), fp32 accumulators; scales meet fp32 numbers only.
//
// Work: the list of all (sequence, kv head, 8 NT rows, 64-token tile) is cut into equal contiguous ranges, one per CTA, at
// least four tiles each; the ranges follow from the lengths on the device.  In a CTA four warps take tiles in turn and
// are joined through shared memory; an item that several CTAs share is joined by the one that draws the last ticket, in
// CTA order.  A CTA shares at most two items (its first and its last), so two slices per CTA are all the scratch there is.
#include "kv_cache.cuh"
#include <algorithm>
#include <cstring>
#include <type_traits>

namespace jgq {

constexpr int KA_WARPS = 4, KA_THREADS = 32 * KA_WARPS;
constexpr int KA_TICKETS = 4096;                       // int32 tickets at the front of the workspace, zero between launches

struct AttendParams {
  const void* q; void* out; float* lse;
  const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
  const int32_t* table; const int32_t* lengths; const int32_t* cu;
  int64_t q_token, q_head;     // strides of q in elements
  int64_t table_stride;
  int32_t* tickets; float* slices;
  int T, B, W, Hq, Hkv, group, D, P, pages;
  int vec_q;                   // 16-byte loads of q are legal
  int zero_rest;               // rows behind the last sequence are zeroed
  int G;                       // CTAs
  float scale;                 // of the scores, times log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x to 2 units in the last place; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_h(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// two codes of a word as f16: as subnormals with their excess, or exact
template <bool EXACT>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int upper) {
  if (!EXACT) return __byte_perm(w, 0u, upper ? 0x4342 : 0x4140);
  uint32_t r = __byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140);         // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__float2half_rn(1152.f)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ int attend_cta_of(int64_t idx, int64_t S, int G) {
  return (int)(((idx + 1) * G + S - 1) / S) - 1;     // the c with c S / G <= idx < (c + 1) S / G
}

__device__ __forceinline__ int seq_rows(const AttendParams& p, int r) {
  if (!p.cu) return 1;
  const int a = max(0, min(p.cu[r], p.T)), b = max(0, min(p.cu[r + 1], p.T));
  return max(0, b - a);
}
__device__ __forceinline__ int seq_len(const AttendParams& p, int r) {
  return (int)min((int64_t)max(0, p.lengths[r]), (int64_t)p.W * p.P);
}

template <typename XT, int DW, int NT>
__global__ void __launch_bounds__(KA_THREADS)
kv_attend_kernel(const AttendParams p) {
  constexpr bool F32 = std::is_same<XT, float>::value;
  constexpr bool EXACT = F32;
  constexpr int QP = F32 ? 2 : 1;                      // planes of q and of p
  constexpr int NC = 8 * NT;                           // rows of q per item
  constexpr int CH = DW / 64;                          // 64-channel chunks of a row
  constexpr int DT = DW / 16;                          // 16-channel tiles of the output
  constexpr int SLICE = NC * (DW + 2);                 // floats: sums, then (max, sum) per row
  constexpr float UP24 = EXACT ? 1.f : 16777216.f;
  extern __shared__ __align__(16) float smem[];        // [warp][NC][DW] sums, [warp][NC][2]
  float* so = smem;
  float* sml = smem + KA_WARPS * NC * DW;
  __shared__ int64_t s_pre[KA_THREADS + 1];
  __shared__ int64_t s_found[2];
  __shared__ int s_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  auto units = [&](int r, int& ct, int& tiles) {       // work of a sequence: kv heads x row tiles x token tiles (one at least)
    const int n = seq_rows(p, r);
    ct = (n * p.group + NC - 1) / NC;
    tiles = n > 0 ? max(1, (seq_len(p, r) + KV_TILE - 1) / KV_TILE) : 0;
    return (int64_t)p.Hkv * ct * tiles;
  };

  // ---- this CTA's range ----
  const int per = (p.B + KA_THREADS - 1) / KA_THREADS;
  {
    int64_t sum = 0;
    int ct, tiles;
    for (int r = tid * per; r < min(p.B, (tid + 1) * per); ++r) sum += units(r, ct, tiles);
    int64_t inc = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_pre[warp] = inc;
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < warp; ++w) before += s_pre[w];
    __syncthreads();
    s_pre[tid + 1] = before + inc;
    if (tid == 0) s_pre[0] = 0;
    __syncthreads();
  }
  const int64_t S = s_pre[KA_THREADS];
  if (p.zero_rest && p.cu) {                           // rows behind the last sequence
    const int64_t first = max(0, min(p.cu[p.B], p.T)), count = (p.T - first) * p.Hq * p.D;
    XT* o = reinterpret_cast<XT*>(p.out) + first * p.Hq * p.D;
    for (int64_t i = blockIdx.x * (int64_t)KA_THREADS + tid; i < count; i += (int64_t)gridDim.x * KA_THREADS) o[i] = from_f32<XT>(0.f);
    if (p.lse)
      for (int64_t i = first * p.Hq + blockIdx.x * (int64_t)KA_THREADS + tid; i < (int64_t)p.T * p.Hq; i += (int64_t)gridDim.x * KA_THREADS) p.lse[i] = -INFINITY;
  }
  const int G = (int)min((int64_t)p.G, (S + KA_WARPS - 1) / KA_WARPS);
  if ((int)blockIdx.x >= G) return;
  const int64_t idx_begin = (int64_t)blockIdx.x * S / G, idx_end = ((int64_t)blockIdx.x + 1) * S / G;
  if (s_pre[tid] <= idx_begin && idx_begin < s_pre[tid + 1]) {
    int64_t at = s_pre[tid];
    int ct, tiles;
    for (int r = tid * per;; ++r) {
      const int64_t u = units(r, ct, tiles);
      if (idx_begin < at + u) { s_found[0] = r; s_found[1] = at; break; }
      at += u;
    }
  }
  __syncthreads();
  int r = (int)s_found[0];
  int64_t seq_at = s_found[1];                         // first unit of the sequence

  // ---- pieces: the part of one item (sequence, head, row tile) in this range ----
  for (int64_t idx = idx_begin; idx < idx_end;) {
    int ct, tiles;
    int64_t u = units(r, ct, tiles);
    while (idx >= seq_at + u) { seq_at += u; ++r; u = units(r, ct, tiles); }
    const int64_t in_seq = idx - seq_at;
    const int item = (int)(in_seq / tiles), h = item / ct, c0 = (item % ct) * NC;
    const int64_t item_at = seq_at + (int64_t)item * tiles;
    const int t_first = (int)(idx - item_at), t_last = (int)min((int64_t)tiles, idx_end - item_at);
    const int n = seq_rows(p, r), L = seq_len(p, r), row_first = p.cu ? max(0, min(p.cu[r], p.T)) : r;
    const int rows = min(NC, n * p.group - c0);        // rows of q of this item
    const int seen_least = max(0, L - n + c0 / p.group + 1);          // what its first row sees

    // ---- q: the lane's operands, and per column (2 t, 2 t + 1 of each octet) limit, factor and sum ----
    uint32_t qf[NT][QP][CH][4][2];
    int limit[NT][2];
    float qscale[NT][2], qbias[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[CH][16], big = 0.f, sum = 0.f;
      const int c = 8 * nt + g, row = c0 + c;
      const bool live = c < rows;
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
        limit[nt][b] = col < rows ? L - n + (c0 + col) / p.group + 1 : 0;
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
    const int32_t* row_of_table = p.table + (int64_t)r * p.table_stride;
    const int tiles_per_page = p.P / KV_TILE;
    const int k_lane = (16 * (g >> 1) + (g & 1)) * DW + 16 * t, v_lane = 64 * g + 16 * t;
    const int t_end = L > 0 ? t_last : t_first;        // a sequence without tokens has one unit and no tile
    for (int tile = t_first + warp; tile < t_end; tile += KA_WARPS) {
      int page = row_of_table[tile / tiles_per_page];
      const bool bad = page < 0 || page >= p.pages;    // no such page: the result is NaN
      if (bad) page = 0;
      const int64_t block = (int64_t)page * p.Hkv + h;
      const int sub = tile % tiles_per_page;
      const uint8_t* kp = p.k + (block * p.P + (int64_t)sub * KV_TILE) * DW + k_lane;
      const uint8_t* vp = p.v + (block * tiles_per_page + sub) * (int64_t)(DW * KV_TILE) + v_lane;
      const float ks = bad ? __int_as_float(0x7fc00000) : p.k_scale[block], vs = p.v_scale[block];

      // scores of 64 tokens: tile i has tokens 16 (g / 2) + 4 i + (g & 1), and those plus two
      float s[4][NT][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][nt][e] = 0.f;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          const uint4 wa = load16(kp + 4 * i * DW + 64 * ch), wb = load16(kp + (4 * i + 2) * DW + 64 * ch);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = code_pair<EXACT>(word_of(wa, j), 0), a2 = code_pair<EXACT>(word_of(wa, j), 1);
            const uint32_t a1 = code_pair<EXACT>(word_of(wb, j), 0), a3 = code_pair<EXACT>(word_of(wb, j), 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int pl = 0; pl < QP; ++pl) mma_h(s[i][nt], a0, a1, a2, a3, qf[nt][pl][ch][j][0], qf[nt][pl][ch][j][1]);
          }
        }
      }
      const bool masked = (tile + 1) * KV_TILE > seen_least;
      uint32_t pb[4][NT][QP][2];                       // p as operands of the products with the values
      float alpha[NT][2], psum[NT][2], vsc[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = fmaf(s[i][nt][e], qscale[nt][e & 1], qbias[nt][e & 1]) * ks;
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
          m[nt][b] = now;
          top[b] = ref;
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
          l[nt][b] = fmaf(l[nt][b], alpha[nt][b], ones[b]);
          psum[nt][b] = EXACT ? 0.f : -128.f * ones[b];
          vsc[nt][b] = ones[b] == 0.f ? 0.f : vs;      // a row that sees none of the tile takes nothing of it, not even a NaN
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const uint4 wa = load16(vp + d * 1024), wb = load16(vp + d * 1024 + 512);
        float x[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[nt][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = code_pair<EXACT>(word_of(wa, i), 0), a2 = code_pair<EXACT>(word_of(wa, i), 1);
          const uint32_t a1 = code_pair<EXACT>(word_of(wb, i), 0), a3 = code_pair<EXACT>(word_of(wb, i), 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pl = 0; pl < QP; ++pl) mma_h(x[nt], a0, a1, a2, a3, pb[i][nt][pl][0], pb[i][nt][pl][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[d][nt][e] = fmaf(fmaf(x[nt][e], UP24, psum[nt][e & 1]), vsc[nt][e & 1], o[d][nt][e] * alpha[nt][e & 1]);
      }
    }

    // ---- join the warps: columns' sums through shared memory ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int col = 8 * nt + 2 * t + b;
        float* dst = so + (warp * NC + col) * DW;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          dst[16 * d + g] = o[d][nt][b];
          dst[16 * d + 8 + g] = o[d][nt][2 + b];
        }
        if (g == 0) { sml[(warp * NC + col) * 2] = m[nt][b]; sml[(warp * NC + col) * 2 + 1] = l[nt][b]; }
      }
    __syncthreads();
    const bool whole = t_first == 0 && t_last == tiles;
    const int first_c = attend_cta_of(item_at, S, G), last_c = attend_cta_of(item_at + tiles - 1, S, G);
    auto finish = [&](int col, int d, float sum, float mx, float den) {
      const int row = c0 + col, token = row_first + row / p.group, head = h * p.group + row % p.group;
      if (d < p.D) reinterpret_cast<XT*>(p.out)[((int64_t)token * p.Hq + head) * p.D + d] = from_f32<XT>(den == 0.f ? 0.f : sum / den);
      if (d == 0 && p.lse) p.lse[(int64_t)token * p.Hq + head] = den == 0.f ? -INFINITY : (mx + log2f(den)) * 0.6931471805599453f;
    };
    float* slice = p.slices + ((int64_t)blockIdx.x * 2 + (idx_begin >= item_at ? 0 : 1)) * SLICE;
    for (int i = tid; i < rows * DW; i += KA_THREADS) {
      const int col = i / DW, d = i % DW;
      float mx = -INFINITY, sum = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) mx = fmaxf(mx, sml[(w * NC + col) * 2]);
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) {
        const float f = exp2_fast(sml[(w * NC + col) * 2] - ref);
        sum = fmaf(so[(w * NC + col) * DW + d], f, sum);
        den = fmaf(sml[(w * NC + col) * 2 + 1], f, den);
      }
      if (whole) {
        finish(col, d, sum, mx, den);
      } else {
        slice[col * DW + d] = sum;
        if (d == 0) { slice[NC * DW + 2 * col] = mx; slice[NC * DW + 2 * col + 1] = den; }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int old = atomicAdd(&p.tickets[first_c], 1);
        s_flag = old == last_c - first_c;
        if (s_flag) p.tickets[first_c] = 0;            // ready for the next launch
      }
      __syncthreads();
      if (s_flag) {
        __threadfence();
        for (int i = tid; i < rows * DW; i += KA_THREADS) {
          const int col = i / DW, d = i % DW;
          float mx = -INFINITY, sum = 0.f, den = 0.f;
          for (int c = first_c; c <= last_c; ++c) {    // in CTA order
            const int64_t begins = (int64_t)c * S / G;
            const float* src = p.slices + ((int64_t)c * 2 + (begins >= item_at ? 0 : 1)) * SLICE;
            const float v = __ldcg(src + NC * DW + 2 * col), dv = __ldcg(src + NC * DW + 2 * col + 1), sv = __ldcg(src + col * DW + d);
            const float now = fmaxf(mx, v), ref = now == -INFINITY ? 0.f : now;
            const float fo = exp2_fast(mx - ref), fn = exp2_fast(v - ref);
            sum = fmaf(sum, fo, sv * fn);
            den = fmaf(den, fo, dv * fn);
            mx = now;
          }
          finish(col, d, sum, mx, den);
        }
      }
    }
    __syncthreads();
    idx = item_at + t_last;
  }
}

// ------------------------------------------------------------------ host ----
struct AttendPlan { int nt, G, smem; size_t slice_bytes; };

static AttendPlan plan_attend(int64_t max_new, int64_t group, int dw, int x_dtype) {
  AttendPlan pl;
  const int64_t rows = max_new * group;
  pl.nt = (rows <= 8 || dw == 256 || x_dtype == JGQ_F32) ? 1 : 2;
  const int nc = 8 * pl.nt;
  pl.smem = KA_WARPS * nc * (dw + 2) * (int)sizeof(float);
  pl.G = std::min(KA_TICKETS, 3 * sm_count());
  pl.slice_bytes = align_up((size_t)pl.G * 2 * nc * (dw + 2) * sizeof(float), 256);
  return pl;
}

template <typename XT, int DW, int NT>
static int launch_attend_inst(const AttendPlan& pl, const AttendParams& p, cudaStream_t s) {
  auto kern = kv_attend_kernel<XT, DW, NT>;
  struct AttrTag {};
  const int arc = once_per_device<AttrTag>([&]() { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, pl.smem); });
  if (arc != 0) return fail(JGQ_ERR_CUDA, "kv_attend: cannot raise the dynamic shared memory limit");
  kern<<<(unsigned)pl.G, KA_THREADS, pl.smem, s>>>(p);
  return check_launch("kv_attend");
}

template <typename XT>
static int launch_attend(const AttendPlan& pl, const AttendParams& p, int dw, cudaStream_t s) {
  constexpr bool F32 = std::is_same<XT, float>::value;
  if (dw == 64) {
    if constexpr (!F32) { if (pl.nt == 2) return launch_attend_inst<XT, 64, 2>(pl, p, s); }
    return launch_attend_inst<XT, 64, 1>(pl, p, s);
  }
  if (dw == 128) {
    if constexpr (!F32) { if (pl.nt == 2) return launch_attend_inst<XT, 128, 2>(pl, p, s); }
    return launch_attend_inst<XT, 128, 1>(pl, p, s);
  }
  return launch_attend_inst<XT, 256, 1>(pl, p, s);
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
  JGQ_REQUIRE(tokens <= (1 << 24) && requests <= (1 << 20) && q_heads <= 4096 && pages <= 2147483647LL && table_width * page_size <= 2147483647LL - 64,
              JGQ_ERR_LIMIT, "kv_attend: shape too large");
  if (tokens == 0) return JGQ_OK;
  JGQ_REQUIRE(q && out && k && v && k_scale && v_scale && lengths && (block_table || table_width == 0), JGQ_ERR_ARG, "kv_attend: null pointer");
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
  p.zero_rest = (flags & JGQ_KV_ZERO_REST) != 0;
  p.G = pl.G;
  p.scale = scale * 1.4426950408889634f;
  cudaStream_t s = (cudaStream_t)stream;
  if (q_dtype == JGQ_F32) return launch_attend<float>(pl, p, dw, s);
  if (q_dtype == JGQ_F16) return launch_attend<__half>(pl, p, dw, s);
  return launch_attend<__nv_bfloat16>(pl, p, dw, s);
}
