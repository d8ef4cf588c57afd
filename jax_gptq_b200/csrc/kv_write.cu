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
// HBM-bound: one CTA per run of rows in a page, head and K or V, one pass: a thread keeps 4 tokens x 16 channels in
// registers between the maximum and the codes.  Neighbouring threads have neighbouring channels for keys (a row's codes are
// contiguous) and neighbouring tokens for values (a channel's are); either way a thread's 16 channels fill 32-byte sectors of the
// rows and its stores complete ones, without shared memory.
// A CTA looks through `chunk` rows for the runs that begin there: few rows per CTA when there are few rows.
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

// The codes of four elements, in excess 128, as a word.  rne(x / s) with the quotient rounded to fp32 is rne(x * (1 / s)) unless
// the product comes within 1e-4 of half way between two whole numbers (its error is below 2e-5): those, and what is not
// finite, are divided.
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float s, float inv) {
  uint32_t b[4];
  bool plain = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = x[i] * inv, t = q + 12582912.f;            // 1.5 * 2^23: the sum's low byte is the rounded q
    const float off = fabsf(q - (t - 12582912.f));
    plain = plain && fabsf(q) <= 127.4f && fabsf(off - 0.5f) >= 1e-4f;
    b[i] = __float_as_uint(t);
  }
  if (!plain) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = x[i] != x[i] ? 0.f : x[i];
      b[i] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.f), 127.f);
    }
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) ^ 0x80808080u;
}

template <typename XT, int DW>
__global__ void __launch_bounds__(KW_MAX_THREADS) kv_write_kernel(const WriteParams p) {
  constexpr int CG = DW / 16;                              // channel groups of a row
  __shared__ float s_top[KW_MAX_THREADS / 32];
  __shared__ uint32_t s_begin[2];
  __shared__ int s_len;
  const int tid = threadIdx.x, h = blockIdx.y, kv = blockIdx.z, P = p.P, threads = blockDim.x;
  const int items = P / 4 * CG;                            // four tokens x 16 channels each
  const bool vec = (kv ? p.vec[1] : p.vec[0]) != 0;
  const int64_t ts = kv ? p.token_stride[1] : p.token_stride[0];
  const XT* x = reinterpret_cast<const XT*>(kv ? p.x[1] : p.x[0]) + h * (kv ? p.head_stride[1] : p.head_stride[0]);
  uint8_t* codes = kv ? p.codes[1] : p.codes[0];
  float* scales = kv ? p.scale[1] : p.scale[0];
  const int64_t limit = p.pages * P, t0 = (int64_t)blockIdx.x * p.chunk;

  // ---- rows of the chunk that begin a run ----
  if (tid < 64) {
    bool begins = false;
    if (tid < p.chunk && t0 + tid < p.T) {
      const int64_t slot = p.slots[t0 + tid];
      begins = slot >= 0 && slot < limit && (slot % P == 0 || t0 + tid == 0 || p.slots[t0 + tid - 1] != slot - 1);
    }
    const uint32_t m = __ballot_sync(0xffffffffu, begins);
    if ((tid & 31) == 0) s_begin[tid >> 5] = m;
  }
  __syncthreads();
  uint64_t todo = s_begin[0] | ((uint64_t)s_begin[1] << 32);
  while (todo) {
    const int64_t t = t0 + __ffsll((long long)todo) - 1;
    todo &= todo - 1;
    const int64_t slot = p.slots[t], page = slot / P;
    const int offset = (int)(slot % P);
    float* scale_at = scales + page * p.H + h;
    const float old = *scale_at;
    // ---- the run: rows t .. t + len - 1 ----
    int len = 1;
    if (t + 1 < p.T && offset + 1 < P && p.slots[t + 1] == slot + 1) {
      if (tid == 0) s_len = (int)min((int64_t)(P - offset), p.T - t);
      __syncthreads();
      for (int i = 1 + tid; i < P - offset && t + i < p.T; i += threads)
        if (p.slots[t + i] != slot + i) { atomicMin(&s_len, i); break; }
      __syncthreads();
      len = s_len;
    }

    Row16<XT> raw[4];
    auto place = [&](int item, int& pos, int& d0) {        // first of the item's four positions in the page, and its channel
      const int quads = P / 4;
      pos = 4 * (kv ? item % quads : item / CG);
      d0 = 16 * (kv ? item / quads : item % CG);
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
    float top = 0.f;
    for (int item = tid; item < items; item += threads) {
      int pos, d0;
      place(item, pos, d0);
      if (pos + 4 > offset && pos < offset + len) {
        fetch(pos, d0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float a = fabsf(row_element<XT>(raw[i], e));
            if (a <= 3.402823466e38f) top = fmaxf(top, a);
          }
      }
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) s_top[tid >> 5] = top;
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) top = fmaxf(top, s_top[w]);
    const float need = __fdiv_rn(top, 127.f);
    const bool begins = offset == 0 || !(old > 0.f);
    float s = begins ? need : old;
    int grown = 0;
    while (s < need && grown < 300) { s *= 2.f; ++grown; }
    uint8_t* base = codes + (page * p.H + h) * (int64_t)P * DW;
    if (grown > 0) {
      const float f = __uint_as_float((uint32_t)(127 - min(grown, 30)) << 23);        // 2^-grown; from 8 on every code becomes 0
      for (int i = tid; i < P * DW / 16; i += threads) {
        uint4 w = reinterpret_cast<const uint4*>(base)[i];
        auto requantized = [&](uint32_t v) {
          uint32_t r = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) r |= (uint32_t)(__float2int_rn((float)((int)((v >> (8 * b)) & 255u) - 128) * f) + 128) << (8 * b);
          return r;
        };
        reinterpret_cast<uint4*>(base)[i] = make_uint4(requantized(w.x), requantized(w.y), requantized(w.z), requantized(w.w));
      }
      __syncthreads();
    }
    if (tid == 0) *scale_at = s;
    const float by = s > 0.f ? s : 1.f, inv = __fdiv_rn(1.f, by);

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
              c[j] = encode4(v, by, inv);
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
          const uint32_t c = encode4(v, by, inv);
          if (all) {
            *reinterpret_cast<uint32_t*>(dst + e * KV_TILE) = c;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pos + i >= offset && pos + i < offset + len) dst[e * KV_TILE + i] = (uint8_t)(c >> (8 * i));
          }
        }
      }
    }
    __syncthreads();
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
  const dim3 grid((unsigned)cdiv(p.T, p.chunk), (unsigned)p.H, 2);
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
  // rows looked through by a CTA: one while that makes no more than some thousand CTAs, up to a tile's 64
  p.chunk = 1;
  while (p.chunk < KV_TILE && cdiv(tokens, p.chunk) * kv_heads * 2 > 4096) p.chunk *= 2;
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
