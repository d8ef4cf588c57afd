// New keys and values into the paged 8-bit cache, and pages back out of it (layout: kv_cache.cuh).
//
// Write.  Row t goes to token slot slots[t] = page * P + offset (negative: nowhere).  The rows of one page and head in
// a call - consecutive rows with ascending slots - are quantized together:
//   need = max |x| / 127                 (finite elements; the quotient rounded to fp32)
//   the page begins (offset 0 is written, or its scale is not positive):  S = need
//   else S = S 2^i, the smallest i >= 0 with S >= need; the codes that are there become rne(code / 2^i)
//   code = rne(x / S) limited to [-127, 127]   (the quotient rounded to fp32; NaN: 0; S = 0: 0)
// Growing by powers of two keeps what a token loses when its page's scale grows below one step of the final scale,
// however often it grows: 1/2 + 1/4 + ... of it on top of nothing but the first rounding's half step.
//
// HBM-bound: a CTA takes a run of rows in a page for a head's keys or values after the other, in one pass each: a thread keeps 4 tokens x 16 channels in
// registers between the maximum and the codes.  Neighbouring threads have neighbouring channels for keys (a row's codes are
// contiguous) and neighbouring tokens for values (a channel's are); either way a thread's 16 channels fill 32-byte sectors of the
// rows and its stores complete ones, without shared memory.
// A CTA looks through `chunk` rows for the runs that begin there; which rows follow on their predecessors is found once, as a
// mask, for the chunk and what its last run may reach.  Runs of one row (a decode step) go to a warp each, without a barrier.
//
// Measured (f16, 32 heads of 128, 6 x 2000 rows into pages of 128): write 107 us (295 MB, 2.7 TB/s), read 76 (302 MB, 4.0 TB/s; 56 behind the write).  A CTA
// loads, takes the maximum and encodes one run after the other, with nothing of the next one under way: a capture of the write shows the wait for
// loads as the first stall, issue 64 %, ALU 54 % (20 instructions per element), and 18 % of the cycles idle at the end.  256 single rows of 8
// heads, bf16: write 9.4 us (1.6 MB: launch and one chain of load, maximum, codes), read of their pages 21; both 30 (49 with IEEE divisions and a CTA per row).
#include "kv_cache.cuh"
#include <algorithm>
#include <cstring>
#include <type_traits>

namespace jgq {

constexpr int KW_MAX_THREADS = 512;

struct WriteParams {
  const void* x[2];            // keys, values
  int64_t token_stride[2], head_stride[2];       // elements
  uint8_t* codes[2]; float* scale[2];
  const int64_t* slots;
  int64_t T, pages;
  int H, D, P, chunk;
  int vec[2];                  // 8 elements at a time are legal
};

// 16 elements of a row, eight or one at a time, as they lie in memory; zeros behind the head dimension
template <typename XT> struct Row16 { uint4 v[sizeof(XT)]; };
template <typename XT>
__device__ __forceinline__ void load_row16(Row16<XT>& r, const XT* src, int left, bool vec) {
  if (vec) {                   // the head dimension is a multiple of 8
#pragma unroll
    for (int i = 0; i < (int)sizeof(XT); ++i)
      r.v[i] = i * (16 / (int)sizeof(XT)) < left ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
  } else {
    XT e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = i < left ? src[i] : from_f32<XT>(0.f);
#pragma unroll
    for (int i = 0; i < (int)sizeof(XT); ++i) {
      constexpr int PER = 16 / (int)sizeof(XT);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(XT) == 4) w[j] = __float_as_uint(to_f32<XT>(e[i * PER + j]));
        else w[j] = (uint32_t)*reinterpret_cast<const uint16_t*>(&e[i * PER + 2 * j]) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&e[i * PER + 2 * j + 1]) << 16);
      }
      r.v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
template <typename XT>
__device__ __forceinline__ float row_element(const Row16<XT>& r, int i) {      // i: known when the code is compiled
  constexpr int PER = 16 / (int)sizeof(XT);
  const uint4 v = r.v[i / PER];
  const int w = (i % PER) * (int)sizeof(XT) / 4;
  const uint32_t u = w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
  if constexpr (std::is_same<XT, float>::value) return __uint_as_float(u);
  else if constexpr (std::is_same<XT, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  else {
    const __half2 h = *reinterpret_cast<const __half2*>(&u);
    return i & 1 ? __high2float(h) : __low2float(h);
  }
}

// The codes of four elements, in excess 128, as a word: rne(x / s) with the quotient rounded to fp32.  x times a reciprocal
// 2^-21 too small and one as much too large, each rounded to a whole number by adding 1.5 * 2^23 (one fused operation, the sum's
// low byte is the number): where both give the same, the quotient and its rounding to fp32, which lie between, do too.
// Otherwise, and where elements are not finite or the reciprocal is not normal (`divide`), the elements are divided.
static __device__ __noinline__ uint32_t encode4_divided(float x0, float x1, float x2, float x3, float s) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = x[i] != x[i] ? 0.f : x[i];
    r |= ((uint32_t)(int)(fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.f), 127.f) + 128.f) & 255u) << (8 * i);
  }
  return r;
}
// bytes a .. b - 1 of a word
static __device__ __noinline__ void store_bytes(uint8_t* dst, uint32_t c, int a, int b) {
  for (int i = a; i < b; ++i) dst[i] = (uint8_t)(c >> (8 * i));
}
struct Reciprocal { float s, lo, hi; uint32_t divide; };
__device__ __forceinline__ Reciprocal reciprocal(float s, bool finite) {
  Reciprocal r;
  r.s = s > 0.f ? s : 1.f;
  const float inv = __fdiv_rn(1.f, r.s);
  const bool ok = finite && r.s >= 1.1754943508222875e-38f && inv >= 1.1754943508222875e-38f;
  r.lo = inv * 0.99999952316284180f;
  r.hi = inv * 1.0000004768371582f;
  r.divide = ok ? 0u : 1u;                               // two NaN of such elements would pass for a quotient
  return r;
}
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], const Reciprocal& q) {
  uint32_t b[4], differ = q.divide;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = __float_as_uint(fmaf(x[i], q.lo, 12582912.f));
    differ |= b[i] ^ __float_as_uint(fmaf(x[i], q.hi, 12582912.f));
  }
  if (differ) return encode4_divided(x[0], x[1], x[2], x[3], q.s);
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) ^ 0x80808080u;
}

// The largest magnitude among four rows' elements: of their bits, two at a time for 16-bit types.  What is not finite comes out
// on top; it is then looked for again among the finite ones.
template <typename XT>
__device__ __forceinline__ uint32_t top_bits(const Row16<XT>& r, uint32_t top) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(XT); ++i) {
    const uint32_t w[4] = {r.v[i].x, r.v[i].y, r.v[i].z, r.v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (sizeof(XT) == 4) top = max(top, w[j] & 0x7fffffffu);
      else asm("max.u16x2 %0, %0, %1;" : "+r"(top) : "r"(w[j] & 0x7fff7fffu));
    }
  }
  return top;
}
template <typename XT>
__device__ __forceinline__ float top_value(uint32_t bits) {            // of the bits of one element, or of two
  if constexpr (sizeof(XT) == 4) return __uint_as_float(bits);
  else {
    const uint16_t b = (uint16_t)max(bits & 0xffffu, bits >> 16);
    return to_f32<XT>(*reinterpret_cast<const XT*>(&b));
  }
}

// scale of a page for rows whose largest magnitude is `top`, and by how many powers of two it has grown
__device__ __forceinline__ float page_scale(float old, float top, bool first, int& grown) {
  const float need = __fdiv_rn(top, 127.f);
  float s = first || !(old > 0.f) ? need : old;
  grown = 0;
  while (s < need && grown < 300) { s *= 2.f; ++grown; }
  return s;
}
// the codes of a page, `bytes` of them, rounded to a scale 2^grown times as large
__device__ __forceinline__ void requantize(uint8_t* base, int bytes, int grown, int thread, int threads) {
  const float f = __uint_as_float((uint32_t)(127 - min(grown, 30)) << 23);            // from 8 on every code becomes 0
  auto word = [&](uint32_t v) {
    uint32_t r = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) r |= (uint32_t)(__float2int_rn((float)((int)((v >> (8 * b)) & 255u) - 128) * f) + 128) << (8 * b);
    return r;
  };
#pragma unroll 4
  for (int i = thread; i < bytes / 16; i += threads) {
    const uint4 w = reinterpret_cast<const uint4*>(base)[i];
    reinterpret_cast<uint4*>(base)[i] = make_uint4(word(w.x), word(w.y), word(w.z), word(w.w));
  }
}

template <typename XT, int DW>
__global__ void __launch_bounds__(KW_MAX_THREADS, sizeof(XT) == 4 ? 1 : 2) kv_write_kernel(const WriteParams p) {
  constexpr int CG = DW / 16;                              // channel groups of a row
  constexpr int MASK = (KV_TILE + 256) / 32;               // words: a chunk and the longest run behind it
  __shared__ float s_top[KW_MAX_THREADS / 32];
  __shared__ uint32_t s_follows[MASK], s_valid[KV_TILE / 32];
  const int tid = threadIdx.x, lane = tid & 31, P = p.P, threads = blockDim.x;
  const int page_shift = P == 64 ? 6 : P == 128 ? 7 : 8;
  const int items = P / 4 * CG;                            // four tokens x 16 channels each
  const int64_t limit = p.pages * P, t0 = (int64_t)blockIdx.x * p.chunk;

  // ---- which rows follow on their predecessor in its page ----
  for (int i = tid; i < MASK * 32; i += threads) {
    bool follows = false, valid = false;
    const int64_t t = t0 + i;
    if (i < p.chunk + P && t < p.T) {
      const int64_t slot = p.slots[t];
      valid = slot >= 0 && slot < limit;
      follows = valid && t > 0 && (slot & (P - 1)) != 0 && p.slots[t - 1] == slot - 1;
    }
    const uint32_t f = __ballot_sync(0xffffffffu, follows), v = __ballot_sync(0xffffffffu, valid);
    if (lane == 0) {
      s_follows[i >> 5] = f;
      if (i < KV_TILE) s_valid[i >> 5] = v;
    }
  }
  __syncthreads();
  const uint64_t in_chunk = p.chunk == 64 ? ~0ull : (1ull << p.chunk) - 1;
  const uint64_t begin = (s_valid[0] | ((uint64_t)s_valid[1] << 32)) & ~(s_follows[0] | ((uint64_t)s_follows[1] << 32)) & in_chunk;
  const uint64_t next_follows = ((s_follows[0] | ((uint64_t)s_follows[1] << 32)) >> 1) | ((uint64_t)(s_follows[2] & 1u) << 63);

  for (int part = blockIdx.y; part < 2 * p.H; part += gridDim.y) {         // keys, then values, of every head
    const int h = part >> 1, kv = part & 1;
    const bool vec = (kv ? p.vec[1] : p.vec[0]) != 0;
    const int64_t ts = kv ? p.token_stride[1] : p.token_stride[0];
    const XT* x = reinterpret_cast<const XT*>(kv ? p.x[1] : p.x[0]) + h * (kv ? p.head_stride[1] : p.head_stride[0]);
    uint8_t* codes = kv ? p.codes[1] : p.codes[0];
    float* scales = kv ? p.scale[1] : p.scale[0];

    // ---- single rows, a warp each ----
    uint64_t todo = begin & ~next_follows;
    for (int n = 0; todo; ++n) {
      const int i = __ffsll((long long)todo) - 1;
      todo &= todo - 1;
      if (n % (threads / 32) != tid / 32) continue;
      constexpr int CPL = DW / 32;                           // channels per lane
      const XT* row = x + (t0 + i) * ts;
      const int d0 = lane * CPL;
      float f[CPL], top = 0.f;
      if (vec && d0 + CPL <= p.D) {
        using V = typename std::conditional<sizeof(XT) * CPL == 32, uint4, typename std::conditional<sizeof(XT) * CPL == 16, uint4,
                  typename std::conditional<sizeof(XT) * CPL == 8, uint2, uint32_t>::type>::type>::type;
        __align__(16) XT e[CPL];
#pragma unroll
        for (int j = 0; j < (int)(sizeof(XT) * CPL / sizeof(V)); ++j) reinterpret_cast<V*>(e)[j] = reinterpret_cast<const V*>(row + d0)[j];
#pragma unroll
        for (int j = 0; j < CPL; ++j) f[j] = to_f32<XT>(e[j]);
      } else {
#pragma unroll
        for (int j = 0; j < CPL; ++j) f[j] = d0 + j < p.D ? to_f32<XT>(row[d0 + j]) : 0.f;
      }
      const int64_t slot = p.slots[t0 + i], page = slot >> page_shift;
      const int offset = (int)slot & (P - 1);
      float* scale_at = scales + page * p.H + h;
      const float old = *scale_at;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const float a = fabsf(f[j]);
        if (a <= 3.402823466e38f) top = fmaxf(top, a);
      }
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      int grown;
      const float s = page_scale(old, top, offset == 0, grown);
      uint8_t* base = codes + (page * p.H + h) * (int64_t)P * DW;
      if (grown > 0) { requantize(base, P * DW, grown, lane, 32); __syncwarp(); }
      if (lane == 0 && (grown > 0 || s != old)) *scale_at = s;
      const Reciprocal by = reciprocal(s, false);            // few elements: divided
#pragma unroll
      for (int j = 0; j < CPL; j += 4) {
        const float v[4] = {f[j], f[j + 1], CPL > 2 ? f[CPL > 2 ? j + 2 : 0] : 0.f, CPL > 2 ? f[CPL > 2 ? j + 3 : 0] : 0.f};
        const uint32_t c = encode4_divided(v[0], v[1], v[2], v[3], by.s);
        if (kv == 0) {
          uint8_t* dst = base + offset * DW + d0 + j;
          if (CPL == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)c;
          else *reinterpret_cast<uint32_t*>(dst) = c;
        } else {
          uint8_t* dst = base + (offset / KV_TILE) * DW * KV_TILE + (d0 + j) * KV_TILE + offset % KV_TILE;
#pragma unroll
          for (int b = 0; b < (CPL < 4 ? CPL : 4); ++b) dst[b * KV_TILE] = (uint8_t)(c >> (8 * b));
        }
      }
    }

    // ---- longer runs, the whole CTA ----
    todo = begin & next_follows;
    while (todo) {
      const int first = __ffsll((long long)todo) - 1;
      todo &= todo - 1;
      const int64_t t = t0 + first, slot = p.slots[t], page = slot >> page_shift;
      const int offset = (int)slot & (P - 1);
      float* scale_at = scales + page * p.H + h;
      const float old = *scale_at;
      int len = 1;                                           // rows t .. t + len - 1
      for (int i = first + 1; i < MASK * 32;) {
        const uint32_t rest = ~(s_follows[i >> 5] >> (i & 31));      // the first row that does not follow
        const int n = rest ? __ffs(rest) - 1 : 32, room = 32 - (i & 31);
        len += min(n, room);
        if (n < room) break;
        i += room;
      }
      len = min(len, P - offset);

      Row16<XT> raw[4];
      auto place = [&](int item, int& pos, int& d0) {        // first of the item's four positions in the page, and its channel
        const int quads = P / 4;
        pos = 4 * (kv ? item & (quads - 1) : item / CG);
        d0 = 16 * (kv ? item >> (page_shift - 2) : item % CG);
      };
      auto fetch = [&](int pos, int d0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = pos + i - offset;
          if (row >= 0 && row < len) load_row16<XT>(raw[i], x + (t + row) * ts + d0, p.D - d0, vec);
          else
#pragma unroll
            for (int j = 0; j < (int)sizeof(XT); ++j) raw[i].v[j] = make_uint4(0, 0, 0, 0);
        }
      };
      uint32_t bits = 0;
      for (int item = tid; item < items; item += threads) {
        int pos, d0;
        place(item, pos, d0);
        if (pos + 4 > offset && pos < offset + len) {
          fetch(pos, d0);
#pragma unroll
          for (int i = 0; i < 4; ++i) bits = top_bits<XT>(raw[i], bits);
        }
      }
      float top = top_value<XT>(bits);
      bool finite = top <= 3.402823466e38f;
      if (!__syncthreads_and(finite)) {
        top = 0.f;
        finite = false;
#pragma unroll 1
        for (int item = tid; item < items; item += threads) {
          int pos, d0;
          place(item, pos, d0);
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            const int row = pos + i - offset;
            if (row < 0 || row >= len) continue;
            for (int e = 0; e < 16 && d0 + e < p.D; ++e) {
              const float a = fabsf(to_f32<XT>(x[(t + row) * ts + d0 + e]));
              if (a <= 3.402823466e38f) top = fmaxf(top, a);
            }
          }
        }
      }
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) s_top[tid >> 5] = top;
      __syncthreads();
      for (int w = 0; w < threads / 32; ++w) top = fmaxf(top, s_top[w]);
      int grown;
      const float s = page_scale(old, top, offset == 0, grown);
      uint8_t* base = codes + (page * p.H + h) * (int64_t)P * DW;
      if (grown > 0) {
        requantize(base, P * DW, grown, tid, threads);
        __syncthreads();
      }
      if (tid == 0) *scale_at = s;
      const Reciprocal by = reciprocal(s, finite);

      for (int item = tid; item < items; item += threads) {
        int pos, d0;
        place(item, pos, d0);
        if (pos + 4 <= offset || pos >= offset + len) continue;
        if (items > threads) fetch(pos, d0);                 // one item per thread is still there
        if (kv == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = pos + i - offset;
            if (row >= 0 && row < len) {
              uint32_t c[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float v[4] = {row_element<XT>(raw[i], 4 * j), row_element<XT>(raw[i], 4 * j + 1), row_element<XT>(raw[i], 4 * j + 2), row_element<XT>(raw[i], 4 * j + 3)};
                c[j] = encode4(v, by);
              }
              *reinterpret_cast<uint4*>(base + (pos + i) * DW + d0) = make_uint4(c[0], c[1], c[2], c[3]);
            }
          }
        } else {
          uint8_t* dst = base + (pos / KV_TILE) * DW * KV_TILE + d0 * KV_TILE + pos % KV_TILE;
          const bool all = pos >= offset && pos + 4 <= offset + len;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float v[4] = {row_element<XT>(raw[0], e), row_element<XT>(raw[1], e), row_element<XT>(raw[2], e), row_element<XT>(raw[3], e)};
            const uint32_t c = encode4(v, by);
            if (all) *reinterpret_cast<uint32_t*>(dst + e * KV_TILE) = c;
            else     store_bytes(dst + e * KV_TILE, c, max(0, offset - pos), min(4, offset + len - pos));
          }
        }
      }
      __syncthreads();
    }
  }
}

// pages[i] -> out[i][head][token][D], keys (z = 0) and values (z = 1); 64 tokens per CTA, 4 x 16 elements per thread as above
struct ReadParams {
  const uint8_t* codes[2]; const float* scale[2]; void* out[2];
  const int64_t* index;
  int64_t pages;
  int H, D, P, vec;
};

template <typename XT, int DW>
__global__ void __launch_bounds__(DW) kv_read_kernel(const ReadParams p) {
  constexpr int CG = DW / 16;
  const int tid = threadIdx.x, kv = blockIdx.z, tiles = p.P / KV_TILE;
  const int64_t item = blockIdx.x / tiles;
  const int sub = blockIdx.x % tiles, h = blockIdx.y;
  const int64_t page = p.index[item];
  const bool bad = page < 0 || page >= p.pages;
  const int64_t block = (bad ? 0 : page) * p.H + h;
  const float s = bad ? __int_as_float(0x7fc00000) : (kv ? p.scale[1] : p.scale[0])[block];
  const uint8_t* src = (kv ? p.codes[1] : p.codes[0]) + (block * tiles + sub) * (int64_t)(DW * KV_TILE);
  const int pos = 4 * (kv ? tid % 16 : tid / CG), d0 = 16 * (kv ? tid / 16 : tid % CG);
  uint32_t c[4][4];                                        // [token][four channels]
  if (kv == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + (pos + i) * DW + d0);
      c[i][0] = v.x; c[i][1] = v.y; c[i][2] = v.z; c[i][3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];                                       // [channel] four tokens
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(src + (d0 + 4 * j + e) * KV_TILE + pos);
      const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);      // tokens 0, 1 of two channels
      const uint32_t e = __byte_perm(w[0], w[1], 0x7362), f = __byte_perm(w[2], w[3], 0x7362);      // tokens 2, 3
      c[0][j] = __byte_perm(a, b, 0x5410); c[1][j] = __byte_perm(a, b, 0x7632);
      c[2][j] = __byte_perm(e, f, 0x5410); c[3][j] = __byte_perm(e, f, 0x7632);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    XT* dst = reinterpret_cast<XT*>(kv ? p.out[1] : p.out[0]) + ((item * p.H + h) * p.P + sub * KV_TILE + pos + i) * (int64_t)p.D + d0;
    __align__(16) XT v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = from_f32<XT>((float)((int)((c[i][e / 4] >> (8 * (e % 4))) & 255u) - 128) * s);
    if (p.vec) {
#pragma unroll
      for (int w = 0; w < (int)sizeof(XT); ++w)
        if (d0 + w * (16 / (int)sizeof(XT)) < p.D) reinterpret_cast<uint4*>(dst)[w] = reinterpret_cast<const uint4*>(v)[w];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (d0 + e < p.D) dst[e] = v[e];
    }
  }
}

template <typename XT>
static int launch_write(const WriteParams& p, int dw, cudaStream_t s) {
  // a CTA takes several heads where that leaves some waves of CTAs: what a chunk's rows are is then found once for them
  const int64_t x = cdiv(p.T, p.chunk);
  const dim3 grid((unsigned)x, (unsigned)std::max<int64_t>(1, std::min<int64_t>(2 * p.H, 32 * (int64_t)sm_count() / x)));
  const int threads = std::min(KW_MAX_THREADS, dw * p.P / KV_TILE);
  if (dw == 64)       kv_write_kernel<XT, 64><<<grid, threads, 0, s>>>(p);
  else if (dw == 128) kv_write_kernel<XT, 128><<<grid, threads, 0, s>>>(p);
  else                kv_write_kernel<XT, 256><<<grid, threads, 0, s>>>(p);
  return check_launch("kv_write");
}

template <typename XT>
static int launch_read(const ReadParams& p, int64_t count, int dw, cudaStream_t s) {
  const dim3 grid((unsigned)(count * (p.P / KV_TILE)), (unsigned)p.H, 2);
  if (dw == 64)       kv_read_kernel<XT, 64><<<grid, 64, 0, s>>>(p);
  else if (dw == 128) kv_read_kernel<XT, 128><<<grid, 128, 0, s>>>(p);
  else                kv_read_kernel<XT, 256><<<grid, 256, 0, s>>>(p);
  return check_launch("kv_read");
}

static int kv_check(const char* what, int dtype, int64_t heads, int64_t head_dim, int64_t pages, int page_size) {
  JGQ_REQUIRE(dtype == JGQ_F32 || dtype == JGQ_F16 || dtype == JGQ_BF16, JGQ_ERR_ARG, "%s: dtype must be f32/f16/bf16", what);
  JGQ_REQUIRE(kv_page_ok(page_size), JGQ_ERR_ARG, "%s: page_size %d is not 64, 128 or 256", what, page_size);
  JGQ_REQUIRE(head_dim >= 1 && head_dim <= 256, JGQ_ERR_ARG, "%s: head_dim %lld not in [1, 256]", what, (long long)head_dim);
  JGQ_REQUIRE(heads >= 1 && pages >= 1, JGQ_ERR_ARG, "%s: bad sizes", what);
  JGQ_REQUIRE(heads <= 4096 && pages <= 2147483647LL, JGQ_ERR_LIMIT, "%s: shape too large", what);
  return JGQ_OK;
}

}  // namespace jgq

using namespace jgq;

extern "C" int jgq_kv_write(const void* k_new, const void* v_new, int dtype, int64_t k_token_stride, int64_t k_head_stride,
                            int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots, int64_t tokens,
                            uint8_t* k, uint8_t* v, float* k_scale, float* v_scale,
                            int64_t pages, int page_size, int64_t kv_heads, int64_t head_dim, void* stream) {
  if (const int rc = kv_check("kv_write", dtype, kv_heads, head_dim, pages, page_size)) return rc;
  JGQ_REQUIRE(tokens >= 0, JGQ_ERR_ARG, "kv_write: bad sizes");
  JGQ_REQUIRE(tokens <= (1 << 24), JGQ_ERR_LIMIT, "kv_write: shape too large");
  if (tokens == 0) return JGQ_OK;
  JGQ_REQUIRE(k_new && v_new && slots && k && v && k_scale && v_scale, JGQ_ERR_ARG, "kv_write: null pointer");
  const size_t xb = dtype_size(dtype);
  JGQ_REQUIRE(aligned(k_new, xb) && aligned(v_new, xb) && aligned(k, 16) && aligned(v, 16) && aligned(slots, 8), JGQ_ERR_ALIGN, "kv_write: misaligned pointer");
  WriteParams p;
  memset(&p, 0, sizeof(p));
  p.x[0] = k_new; p.x[1] = v_new;
  p.token_stride[0] = k_token_stride; p.token_stride[1] = v_token_stride;
  p.head_stride[0] = k_head_stride; p.head_stride[1] = v_head_stride;
  p.codes[0] = k; p.codes[1] = v; p.scale[0] = k_scale; p.scale[1] = v_scale;
  p.slots = slots; p.T = tokens; p.pages = pages;
  p.H = (int)kv_heads; p.D = (int)head_dim; p.P = page_size;
  for (int i = 0; i < 2; ++i)
    p.vec[i] = head_dim % 8 == 0 && aligned(p.x[i], 16) && p.token_stride[i] * xb % 16 == 0 && p.head_stride[i] * xb % 16 == 0;
  // rows looked through by a CTA: two while that makes no more than some thousand CTAs, up to a tile's 64
  p.chunk = 2;
  while (p.chunk < KV_TILE && cdiv(tokens, p.chunk) * kv_heads * 2 > 2048) p.chunk *= 2;
  cudaStream_t s = (cudaStream_t)stream;
  const int dw = kv_width(head_dim);
  if (dtype == JGQ_F32) return launch_write<float>(p, dw, s);
  if (dtype == JGQ_F16) return launch_write<__half>(p, dw, s);
  return launch_write<__nv_bfloat16>(p, dw, s);
}

extern "C" int jgq_kv_read(const uint8_t* k, const uint8_t* v, const float* k_scale, const float* v_scale,
                           int64_t pages, int page_size, int64_t kv_heads, int64_t head_dim,
                           const int64_t* index, int64_t count, void* k_out, void* v_out, int dtype, void* stream) {
  if (const int rc = kv_check("kv_read", dtype, kv_heads, head_dim, pages, page_size)) return rc;
  JGQ_REQUIRE(count >= 0, JGQ_ERR_ARG, "kv_read: bad sizes");
  JGQ_REQUIRE(count * (page_size / KV_TILE) <= 2147483647LL, JGQ_ERR_LIMIT, "kv_read: shape too large");
  if (count == 0) return JGQ_OK;
  JGQ_REQUIRE(k && v && k_scale && v_scale && index && k_out && v_out, JGQ_ERR_ARG, "kv_read: null pointer");
  const size_t xb = dtype_size(dtype);
  JGQ_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_out, xb) && aligned(v_out, xb) && aligned(index, 8), JGQ_ERR_ALIGN, "kv_read: misaligned pointer");
  ReadParams p;
  memset(&p, 0, sizeof(p));
  p.codes[0] = k; p.codes[1] = v; p.scale[0] = k_scale; p.scale[1] = v_scale; p.out[0] = k_out; p.out[1] = v_out;
  p.index = index; p.pages = pages; p.H = (int)kv_heads; p.D = (int)head_dim; p.P = page_size;
  p.vec = head_dim % 8 == 0 && aligned(k_out, 16) && aligned(v_out, 16);
  cudaStream_t s = (cudaStream_t)stream;
  const int dw = kv_width(head_dim);
  if (dtype == JGQ_F32) return launch_read<float>(p, count, dw, s);
  if (dtype == JGQ_F16) return launch_read<__half>(p, count, dw, s);
  return launch_read<__nv_bfloat16>(p, count, dw, s);
}
