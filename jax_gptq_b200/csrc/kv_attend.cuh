// What the attention kernels over the paged cache share: parameters, the cut of the work, small device helpers.
#pragma once
#include "kv_cache.cuh"
#include "umma.cuh"
#include <type_traits>

namespace jgq {

constexpr int KA_TICKETS = 4096;                       // int32 tickets at the front of the workspace, zero between launches

struct AttendParams {
  const void* q; void* out; float* lse;
  const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
  const int32_t* table; const int32_t* lengths; const int32_t* cu;
  int64_t q_token, q_head;     // strides of q in elements
  int64_t table_stride;
  int32_t* tickets; float* slices;
  int T, B, W, Hq, Hkv, group, D, P, pages;
  int q_map;                   // prompts: rows of q come by TMA
  int vec_q, vec_o;            // 16-byte loads of q, stores of four channels are legal
  int zero_rest;               // rows of no sequence are zeroed
  int G;                       // CTAs
  float scale;                 // of the scores, times log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x to 2 units in the last place; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a page's scale of keys: infinity spoils its page's scores as NaN does (it could pass for a token that is masked)
__device__ __forceinline__ float attend_key_scale(float s) { return s + (s - s); }
__device__ __forceinline__ void mma_h(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_h0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // d = a b
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
// An ordinary load: behind the wait that goes before it, but free to move among products and other loads.
__device__ __forceinline__ uint4 lds16(uint32_t at) { return *reinterpret_cast<const uint4*>(__cvta_shared_to_generic(at)); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(umma::smem_u32(bar)) : "memory");
}

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

// sum over i < n of floor((a i + b) / m); a, b >= 0
template <typename T>
__device__ __forceinline__ int64_t floor_sum_of(T n, T m, T a, T b) {
  int64_t sum = 0;
  while (n > 0) {
    if (a >= m) { const T q = a / m; sum += (int64_t)n * (n - 1) / 2 * q; a -= q * m; }
    if (b >= m) { const T q = b / m; sum += (int64_t)n * q; b -= q * m; }
    const T y = a * n + b;
    if (y < m) break;
    n = y / m;                                         // the lattice points below the line, counted along the other axis
    b = y - n * m;
    const T t = a; a = m; m = t;
  }
  return sum;
}
// (quotients of 64 bits take five times as long: 32 where they do; n and m only shrink)
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  return a * n + b < (1ll << 31) && n < 65536 && m < 65536 ? floor_sum_of<uint32_t>((uint32_t)n, (uint32_t)m, (uint32_t)a, (uint32_t)b) : floor_sum_of<int64_t>(n, m, a, b);
}

// a sequence's part of the list: row tiles per head, and units of row tile c: floor((a c + b) / m), COST in front and a tile each
struct SeqWork {
  int n, L, ct;
  int64_t m, a, b;
};
template <int NC, int COST>
__device__ __forceinline__ SeqWork seq_work(const AttendParams& p, int r) {
  SeqWork w;
  w.n = seq_rows(p, r);
  w.L = seq_len(p, r);
  w.ct = (w.n * p.group + NC - 1) / NC;
  w.m = 1; w.a = 0; w.b = COST + max(1, (w.L + KV_TILE - 1) / KV_TILE);
  if (w.ct > 1 && w.L >= w.n) {                        // what the last row of row tile c sees, in tokens times group, rounded up
    w.m = (int64_t)KV_TILE * p.group;
    w.a = NC;
    w.b = (int64_t)(w.L - w.n) * p.group + NC + p.group - 1 + w.m - 1 + COST * w.m;
  }
  return w;
}

template <int NC, int COST>
__device__ __forceinline__ int64_t seq_units(const AttendParams& p, int r) {
  const SeqWork w = seq_work<NC, COST>(p, r);
  return w.n > 0 ? (int64_t)p.Hkv * (w.a ? floor_sum(w.ct, w.m, w.a, w.b) : w.ct * w.b) : 0;
}

// The list of all units cut into equal contiguous ranges, one per CTA, `least` units at least.
struct AttendRange {
  int64_t S, begin, end;       // units in all, this CTA's
  int G;                       // CTAs that have a range; this one if blockIdx.x < G
  int r;                       // the sequence `begin` lies in, and its first unit
  int64_t seq_at;
};
// Every thread sums up a run of consecutive sequences; s_pre: THREADS + 1 words, s_found: 2.
template <int NC, int COST, int THREADS>
__device__ __forceinline__ AttendRange attend_range(const AttendParams& p, int least, int64_t* s_pre, int64_t* s_found) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (p.B + THREADS - 1) / THREADS;
  AttendRange g;
  int64_t sum = 0;
  for (int r = tid * per; r < min(p.B, (tid + 1) * per); ++r) sum += seq_units<NC, COST>(p, r);
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
  g.S = s_pre[THREADS];
  g.G = (int)min((int64_t)p.G, (g.S + least - 1) / least);
  g.begin = g.end = g.seq_at = 0;
  g.r = 0;
  if ((int)blockIdx.x >= g.G) return g;
  g.begin = (int64_t)blockIdx.x * g.S / g.G;
  g.end = ((int64_t)blockIdx.x + 1) * g.S / g.G;
  if (s_pre[tid] <= g.begin && g.begin < s_pre[tid + 1]) {
    int64_t at = s_pre[tid];
    for (int r = tid * per;; ++r) {
      const int64_t u = seq_units<NC, COST>(p, r);
      if (g.begin < at + u) { s_found[0] = r; s_found[1] = at; break; }
      at += u;
    }
  }
  __syncthreads();
  g.r = (int)s_found[0];
  g.seq_at = s_found[1];
  return g;
}

// The piece of the item (sequence, kv head, NC rows of q) at unit idx of a range.
struct AttendPiece {
  int n, L, h, c0, rows;       // rows of the sequence, tokens, kv head, first row of q, rows of q
  int row_first;               // the sequence's first row among all
  int t_first, t_last, tiles;  // tiles of the piece, and of the item
  int64_t tile_at;             // unit of the item's tile 0
};
// Where a range stands: set to its first item, then moved from item to item.
template <int NC, int COST>
struct AttendCursor {
  SeqWork wk;
  int h, row_tile, units;      // item and its units
  int64_t at;                  // its first unit
  int row_first;

  __device__ __forceinline__ void open(const AttendParams& p, const AttendRange& g) {
    wk = seq_work<NC, COST>(p, g.r);
    row_first = p.cu ? max(0, min(p.cu[g.r], p.T)) : g.r;
  }
  __device__ __forceinline__ int units_of(int c) const { return wk.a == 0 ? (int)wk.b : (int)((wk.a * c + wk.b) / wk.m); }
  // whole warps: the lanes look for the row tile together
  __device__ __forceinline__ void find(const AttendParams& p, const AttendRange& g) {
    open(p, g);
    const int64_t per_head = wk.a ? floor_sum(wk.ct, wk.m, wk.a, wk.b) : wk.ct * wk.b;
    h = (int)((g.begin - g.seq_at) / per_head);
    const int64_t in_head = g.begin - g.seq_at - h * per_head;
    int64_t before;
    if (wk.a) {
      int lo = 0, hi = wk.ct;                          // sums up to lo are at most in_head, up to hi more
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, c = min(hi, lo + ((threadIdx.x & 31) + 1) * step);
        const uint32_t m = __ballot_sync(0xffffffffu, c >= hi || floor_sum(c, wk.m, wk.a, wk.b) > in_head);
        const int first = __ffs(m) - 1;                // the last lane's c is hi: there is one
        hi = min(hi, lo + (first + 1) * step);
        lo += first * step;
      }
      row_tile = lo;
      before = floor_sum(lo, wk.m, wk.a, wk.b);
    } else {
      row_tile = (int)(in_head / wk.b);
      before = row_tile * wk.b;
    }
    at = g.seq_at + h * per_head + before;
    units = units_of(row_tile);
  }
  __device__ __forceinline__ void next(const AttendParams& p, AttendRange& g) {
    at += units;
    if (++row_tile == wk.ct) {
      row_tile = 0;
      if (++h == p.Hkv) {
        h = 0;
        do { ++g.r; } while (g.r < p.B && seq_rows(p, g.r) == 0);
        if (g.r < p.B) open(p, g);
      }
    }
    units = units_of(row_tile);
  }
  __device__ __forceinline__ AttendPiece piece(const AttendParams& p, const AttendRange& g, int64_t idx) const {
    AttendPiece e;
    e.n = wk.n; e.L = wk.L; e.h = h;
    e.c0 = row_tile * NC;
    e.rows = min(NC, e.n * p.group - e.c0);
    e.row_first = row_first;
    e.tiles = units - COST;
    e.tile_at = at + COST;
    e.t_first = (int)max((int64_t)0, idx - e.tile_at);
    e.t_last = (int)max((int64_t)0, min((int64_t)e.tiles, g.end - e.tile_at));
    return e;
  }
};

// rows of q behind the last sequence, and in front of the first, become zero
template <typename XT, int THREADS>
__device__ __forceinline__ void attend_zero_rest(const AttendParams& p) {
  if (!p.zero_rest || !p.cu) return;
  const int64_t front = max(0, min(p.cu[0], p.T)), behind = max(0, min(p.cu[p.B], p.T)), at = blockIdx.x * (int64_t)THREADS + threadIdx.x;
  auto clear = [&](int64_t first, int64_t rows) {
    XT* o = reinterpret_cast<XT*>(p.out) + first * p.Hq * p.D;
    for (int64_t i = at; i < rows * p.Hq * p.D; i += (int64_t)gridDim.x * THREADS) o[i] = from_f32<XT>(0.f);
    if (p.lse)
      for (int64_t i = at; i < rows * p.Hq; i += (int64_t)gridDim.x * THREADS) p.lse[first * p.Hq + i] = -INFINITY;
  };
  if (front > 0) clear(0, min(front, behind));
  clear(behind, p.T - behind);
}

// where row `col` of an item goes: the row of (token, head)
__device__ __forceinline__ int64_t attend_out_row(const AttendParams& p, const AttendPiece& e, int col) {
  const int row = e.c0 + col, i = p.group == 1 ? row : row / p.group;
  return (int64_t)(e.row_first + i) * p.Hq + e.h * p.group + (row - i * p.group);
}
__device__ __forceinline__ void attend_put_lse(const AttendParams& p, int64_t at, float mx, float den) {
  if (p.lse) p.lse[at] = den == 0.f ? -INFINITY : (mx + log2f(den)) * 0.6931471805599453f;
}
// four channels of a row's result: sums times f, to row `at` of the output
template <typename XT>
__device__ __forceinline__ void attend_store4(const AttendParams& p, int64_t at, int d, const float4& sum, float f) {
  const float v[4] = {sum.x * f, sum.y * f, sum.z * f, sum.w * f};
  XT* dst = reinterpret_cast<XT*>(p.out) + at * p.D + d;
  if (p.vec_o) {
    if (d < p.D) {
      __align__(16) XT e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = from_f32<XT>(v[i]);
      if constexpr (sizeof(XT) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(e);
      else                           *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.D) dst[i] = from_f32<XT>(v[i]);
  }
}
template <typename XT>
__device__ __forceinline__ void attend_finish4(const AttendParams& p, const AttendPiece& piece, int col, int d, const float4& sum, float mx, float den) {
  const int64_t at = attend_out_row(p, piece, col);
  attend_store4<XT>(p, at, d, sum, den == 0.f ? 0.f : __fdiv_rn(1.f, den));
  if (d == 0) attend_put_lse(p, at, mx, den);
}

// A CTA shares at most two items, its first (the one its range begins inside of) and its last: slice 0 and slice 1.
// A slice holds the sums [NC][DW] relative to the row's maximum, then (maximum, sum of exponentials) per row.
template <int NC, int DW>
__device__ __forceinline__ float* attend_slice(const AttendParams& p, const AttendRange& g, int cta, const AttendPiece& e) {
  return p.slices + ((int64_t)cta * 2 + ((int64_t)cta * g.S / g.G > e.tile_at ? 0 : 1)) * (NC * (DW + 2));
}
// After a CTA's slice of an item is written (all threads): true in the CTA that is the last one; the tickets are left zero.
__device__ __forceinline__ bool attend_last(const AttendParams& p, int first_c, int last_c, int* s_flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int old = atomicAdd(&p.tickets[first_c], 1);
    *s_flag = old == last_c - first_c;
    if (*s_flag) p.tickets[first_c] = 0;               // ready for the next launch
  }
  __syncthreads();
  const bool last = *s_flag != 0;
  if (last) __threadfence();
  return last;
}
// The slices of an item added in CTA order: four channels of JP rows per thread, SL slices at a time: SL JP loads in flight.
template <typename XT, int NC, int DW, int THREADS, int JP, int SL>
__device__ __forceinline__ void attend_join(const AttendParams& p, const AttendRange& g, const AttendPiece& e, int first_c, int last_c) {
  const int count = e.rows * (DW / 4);
  for (int i0 = threadIdx.x; i0 < count; i0 += THREADS * JP) {
    float mx[JP], den[JP];
    float4 sum[JP];
#pragma unroll
    for (int j = 0; j < JP; ++j) { mx[j] = -INFINITY; den[j] = 0.f; sum[j] = make_float4(0.f, 0.f, 0.f, 0.f); }
    for (int cb = first_c; cb <= last_c; cb += SL) {
      float v[SL][JP], dv[SL][JP];
      float4 sv[SL][JP];
#pragma unroll
      for (int c = 0; c < SL; ++c) {
        const float* src = attend_slice<NC, DW>(p, g, min(cb + c, last_c), e);
#pragma unroll
        for (int j = 0; j < JP; ++j) {
          const int i = min(i0 + j * THREADS, count - 1), col = i / (DW / 4);
          v[c][j] = __ldcg(src + NC * DW + 2 * col);
          dv[c][j] = __ldcg(src + NC * DW + 2 * col + 1);
          sv[c][j] = __ldcg(reinterpret_cast<const float4*>(src) + i);
        }
      }
#pragma unroll
      for (int c = 0; c < SL; ++c)
        if (cb + c <= last_c) {
#pragma unroll
          for (int j = 0; j < JP; ++j) {
            const float now = fmaxf(mx[j], v[c][j]), ref = now == -INFINITY ? 0.f : now;
            const float fo = exp2_fast(mx[j] - ref), fn = exp2_fast(v[c][j] - ref);
            sum[j].x = fmaf(sum[j].x, fo, sv[c][j].x * fn); sum[j].y = fmaf(sum[j].y, fo, sv[c][j].y * fn);
            sum[j].z = fmaf(sum[j].z, fo, sv[c][j].z * fn); sum[j].w = fmaf(sum[j].w, fo, sv[c][j].w * fn);
            den[j] = fmaf(den[j], fo, dv[c][j] * fn);
            mx[j] = now;
          }
        }
    }
#pragma unroll
    for (int j = 0; j < JP; ++j) {
      const int i = i0 + j * THREADS;
      if (i < count) attend_finish4<XT>(p, e, i / (DW / 4), 4 * (i % (DW / 4)), sum[j], mx[j], den[j]);
    }
  }
}

// The same for many rows: a thread first finds a row's maximum and sum over all slices, then the sums are added with weights of
// known size.  `at`: the rows' places in the output (shared memory), `ml`, `inv`: room for them.
template <typename XT, int NC, int DW, int THREADS, int JP, int SL>
__device__ __forceinline__ void attend_join_rows(const AttendParams& p, const AttendRange& g, const AttendPiece& e, int first_c, int last_c,
                                                 const int64_t* at, float2* ml, float* inv) {
  __syncthreads();                                     // the rows' places are known, and nothing reads ml and inv any more
  for (int col = threadIdx.x; col < e.rows; col += THREADS) {
    float mx = -INFINITY, den = 0.f;
    for (int cb = first_c; cb <= last_c; cb += SL) {
      float2 v[SL];
#pragma unroll
      for (int c = 0; c < SL; ++c) v[c] = __ldcg(reinterpret_cast<const float2*>(attend_slice<NC, DW>(p, g, min(cb + c, last_c), e) + NC * DW) + col);
#pragma unroll
      for (int c = 0; c < SL; ++c)
        if (cb + c <= last_c) {
          const float now = fmaxf(mx, v[c].x), ref = now == -INFINITY ? 0.f : now;
          den = fmaf(den, exp2_fast(mx - ref), v[c].y * exp2_fast(v[c].x - ref));
          mx = now;
        }
    }
    ml[col] = make_float2(mx == -INFINITY ? 0.f : mx, den);
    inv[col] = den == 0.f ? 0.f : __fdiv_rn(1.f, den);
    if (p.lse) attend_put_lse(p, at[col], mx, den);
  }
  __syncthreads();
  const int count = e.rows * (DW / 4);
  for (int i0 = threadIdx.x; i0 < count; i0 += THREADS * JP) {
    float4 sum[JP];
    float ref[JP];
#pragma unroll
    for (int j = 0; j < JP; ++j) {
      sum[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      ref[j] = ml[min(i0 + j * THREADS, count - 1) / (DW / 4)].x;
    }
    for (int cb = first_c; cb <= last_c; cb += SL) {
      float w[SL][JP];
      float4 sv[SL][JP];
#pragma unroll
      for (int c = 0; c < SL; ++c) {
        const float* src = attend_slice<NC, DW>(p, g, min(cb + c, last_c), e);
#pragma unroll
        for (int j = 0; j < JP; ++j) {
          const int i = min(i0 + j * THREADS, count - 1);
          w[c][j] = __ldcg(src + NC * DW + 2 * (i / (DW / 4)));
          sv[c][j] = __ldcg(reinterpret_cast<const float4*>(src) + i);
        }
      }
#pragma unroll
      for (int c = 0; c < SL; ++c)
        if (cb + c <= last_c) {
#pragma unroll
          for (int j = 0; j < JP; ++j) {
            const float f = exp2_fast(w[c][j] - ref[j]);
            sum[j].x = fmaf(sv[c][j].x, f, sum[j].x); sum[j].y = fmaf(sv[c][j].y, f, sum[j].y);
            sum[j].z = fmaf(sv[c][j].z, f, sum[j].z); sum[j].w = fmaf(sv[c][j].w, f, sum[j].w);
          }
        }
    }
#pragma unroll
    for (int j = 0; j < JP; ++j) {
      const int i = i0 + j * THREADS, col = i / (DW / 4);
      if (i < count) attend_store4<XT>(p, at[col], 4 * (i % (DW / 4)), sum[j], inv[col]);
    }
  }
}

// the prompt kernel (kv_prompt.cu): 256 rows of q per item, 16-bit types, rows of 64 or 128 channels
struct PromptPlan { int use, G; size_t slice_bytes; };
PromptPlan plan_kv_prompt(int64_t rows, int dw, int q_dtype);
int launch_kv_prompt(const PromptPlan& pl, AttendParams& p, int dw, int q_dtype, cudaStream_t s);

}  // namespace jgq
