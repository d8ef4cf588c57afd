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
// HBM-bound: one CTA per run of rows in a page, head and K or V; a run is read twice, the second time out of L1 / L2.
// A CTA looks through `chunk` rows for the runs that begin there: few rows per CTA when there are few rows.
#include "kv_cache.cuh"
#include <algorithm>
#include <cstring>
#include <type_traits>

namespace jgq {

constexpr int KW_THREADS = 128;

struct WriteParams {
  const void* x[2];            // keys, values
  int64_t token_stride[2], head_stride[2];       // elements
  uint8_t* codes[2]; float* scale[2];
  const int64_t* slots;
  int64_t T, pages;
  int H, D, P, chunk;
  int vec[2];                  // 8 elements at a time are legal
};

// eight elements of a row from channel d on; zeros behind the head dimension
template <typename XT>
__device__ __forceinline__ void row8(float (&f)[8], const XT* src, int d, int D, bool vec) {
  if (vec) {                   // D % 8 == 0
    if (d < D) {
      __align__(16) XT e[8];
#pragma unroll
      for (int v = 0; v < (int)sizeof(XT) / 2; ++v) reinterpret_cast<uint4*>(e)[v] = reinterpret_cast<const uint4*>(src + d)[v];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32<XT>(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = d + i < D ? to_f32<XT>(src[d + i]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t encode(float x, float s) {
  if (x != x) x = 0.f;
  return (uint32_t)(int)(fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f) + 128.f);
}

template <typename XT, int DW>
__global__ void __launch_bounds__(KW_THREADS) kv_write_kernel(const WriteParams p) {
  constexpr int TPR = DW / 8, RPP = KW_THREADS / TPR;      // threads per row, rows at a time
  constexpr int VST = KV_TILE + 4;                         // bytes per channel of the transposed tile
  __shared__ __align__(16) uint8_t tile[DW * VST];
  __shared__ float s_top[KW_THREADS / 32];
  __shared__ int s_len;
  const int tid = threadIdx.x, h = blockIdx.y, kv = blockIdx.z, P = p.P;
  const int rt = tid / TPR, d0 = 8 * (tid % TPR);
  const bool vec = p.vec[kv] != 0;
  const XT* x = reinterpret_cast<const XT*>(p.x[kv]) + h * p.head_stride[kv];
  const int64_t ts = p.token_stride[kv], limit = p.pages * P;

  const int64_t t_end = min(p.T, ((int64_t)blockIdx.x + 1) * p.chunk);
  for (int64_t t = (int64_t)blockIdx.x * p.chunk; t < t_end; ++t) {
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= limit) continue;
    const int offset = (int)(slot % P);
    if (t > 0 && offset != 0 && p.slots[t - 1] == slot - 1) continue;        // belongs to the run before
    const int64_t page = slot / P;
    // ---- the run: rows t .. t + len - 1 ----
    if (tid == 0) s_len = (int)min((int64_t)(P - offset), p.T - t);
    __syncthreads();
    for (int i = 1 + tid; i < P - offset && t + i < p.T; i += KW_THREADS)
      if (p.slots[t + i] != slot + i) { atomicMin(&s_len, i); break; }
    __syncthreads();
    const int len = s_len;

    float top = 0.f;
    for (int i = rt; i < len; i += RPP) {
      float f[8];
      row8<XT>(f, x + (t + i) * ts, d0, p.D, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(f[e]);
        if (a <= 3.402823466e38f) top = fmaxf(top, a);
      }
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) s_top[tid >> 5] = top;
    float* scale_at = p.scale[kv] + page * p.H + h;
    const float old = *scale_at;
    __syncthreads();
    for (int w = 0; w < KW_THREADS / 32; ++w) top = fmaxf(top, s_top[w]);
    const float need = __fdiv_rn(top, 127.f);
    const bool begins = offset == 0 || !(old > 0.f);
    float s = begins ? need : old;
    int grown = 0;
    while (s < need && grown < 300) { s *= 2.f; ++grown; }
    uint8_t* base = p.codes[kv] + (page * p.H + h) * (int64_t)P * DW;
    if (grown > 0) {
      const float f = __uint_as_float((uint32_t)(127 - min(grown, 30)) << 23);        // 2^-grown; from 8 on every code becomes 0
      for (int i = tid; i < P * DW / 16; i += KW_THREADS) {
        uint4 w = reinterpret_cast<const uint4*>(base)[i];
        uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            r |= (uint32_t)(__float2int_rn((float)((int)((e[j] >> (8 * b)) & 255u) - 128) * f) + 128) << (8 * b);
          e[j] = r;
        }
        reinterpret_cast<uint4*>(base)[i] = w;
      }
      __syncthreads();
    }
    if (tid == 0) *scale_at = s;
    const float by = s > 0.f ? s : 1.f;

    if (kv == 0) {
      for (int i = rt; i < len; i += RPP) {
        float f[8];
        row8<XT>(f, x + (t + i) * ts, d0, p.D, vec);
        uint32_t c[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e >> 2] |= encode(f[e], by) << (8 * (e & 3));
        *reinterpret_cast<uint2*>(base + (int64_t)(offset + i) * DW + d0) = make_uint2(c[0], c[1]);
      }
    } else if (len < 16) {
      for (int i = rt; i < len; i += RPP) {
        float f[8];
        row8<XT>(f, x + (t + i) * ts, d0, p.D, vec);
        const int at = offset + i;
        uint8_t* dst = base + (int64_t)(at / KV_TILE) * DW * KV_TILE + d0 * KV_TILE + at % KV_TILE;
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e * KV_TILE] = (uint8_t)encode(f[e], by);
      }
    } else {
      // 64 tokens at a time through shared memory, channel by channel
      for (int first = offset / KV_TILE * KV_TILE; first < offset + len; first += KV_TILE) {
        const int a = max(0, offset - first), b = min(KV_TILE, offset + len - first);
        for (int i = a + rt; i < b; i += RPP) {
          float f[8];
          row8<XT>(f, x + (t + first + i - offset) * ts, d0, p.D, vec);
#pragma unroll
          for (int e = 0; e < 8; ++e) tile[(d0 + e) * VST + i] = (uint8_t)encode(f[e], by);
        }
        __syncthreads();
        uint8_t* dst = base + (int64_t)(first / KV_TILE) * DW * KV_TILE;
        for (int i = tid; i < DW * (KV_TILE / 16); i += KW_THREADS) {
          const int d = i / (KV_TILE / 16), c = 16 * (i % (KV_TILE / 16));
          const uint8_t* src = tile + d * VST + c;
          if (c >= a && c + 16 <= b) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
            *reinterpret_cast<uint4*>(dst + d * KV_TILE + c) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
            for (int e = 0; e < 16; ++e)
              if (c + e >= a && c + e < b) dst[d * KV_TILE + c + e] = src[e];
          }
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
}

// pages[i] -> out[i][head][token][D], keys (z = 0) and values (z = 1); 64 tokens per CTA
struct ReadParams {
  const uint8_t* codes[2]; const float* scale[2]; void* out[2];
  const int64_t* index;
  int64_t pages;
  int H, D, P, vec;
};

template <typename XT, int DW>
__global__ void __launch_bounds__(KW_THREADS) kv_read_kernel(const ReadParams p) {
  constexpr int VST = KV_TILE + 4;
  __shared__ __align__(16) uint8_t tile[DW * VST];
  const int tid = threadIdx.x, kv = blockIdx.z, tiles = p.P / KV_TILE;
  const int64_t item = blockIdx.x / tiles;
  const int sub = blockIdx.x % tiles, h = blockIdx.y;
  const int64_t page = p.index[item];
  const bool bad = page < 0 || page >= p.pages;
  const int64_t block = (bad ? 0 : page) * p.H + h;
  const float s = bad ? __int_as_float(0x7fc00000) : p.scale[kv][block];
  const uint8_t* src = p.codes[kv] + (block * tiles + sub) * (int64_t)(DW * KV_TILE);
  XT* dst = reinterpret_cast<XT*>(p.out[kv]) + ((item * p.H + h) * p.P + sub * KV_TILE) * (int64_t)p.D;
  if (kv == 1) {
    for (int i = tid; i < DW * (KV_TILE / 4); i += KW_THREADS)
      *reinterpret_cast<uint32_t*>(tile + (i / (KV_TILE / 4)) * VST + 4 * (i % (KV_TILE / 4))) = reinterpret_cast<const uint32_t*>(src)[i];
    __syncthreads();
  }
  constexpr int TPR = DW / 8;
  for (int i = tid; i < KV_TILE * TPR; i += KW_THREADS) {
    const int r = i / TPR, d0 = 8 * (i % TPR);
    uint32_t c[2];
    if (kv == 0) {
      const uint2 w = *reinterpret_cast<const uint2*>(src + r * DW + d0);
      c[0] = w.x; c[1] = w.y;
    } else {
      c[0] = c[1] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e >> 2] |= (uint32_t)tile[(d0 + e) * VST + r] << (8 * (e & 3));
    }
    __align__(16) XT v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = from_f32<XT>((float)((int)((c[e >> 2] >> (8 * (e & 3))) & 255u) - 128) * s);
    XT* o = dst + (int64_t)r * p.D + d0;
    if (p.vec) {
      if (d0 < p.D)
#pragma unroll
        for (int w = 0; w < (int)sizeof(XT) / 2; ++w) reinterpret_cast<uint4*>(o)[w] = reinterpret_cast<const uint4*>(v)[w];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < p.D) o[e] = v[e];
    }
  }
}

template <typename XT>
static int launch_write(const WriteParams& p, int dw, cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(p.T, p.chunk), (unsigned)p.H, 2);
  if (dw == 64)       kv_write_kernel<XT, 64><<<grid, KW_THREADS, 0, s>>>(p);
  else if (dw == 128) kv_write_kernel<XT, 128><<<grid, KW_THREADS, 0, s>>>(p);
  else                kv_write_kernel<XT, 256><<<grid, KW_THREADS, 0, s>>>(p);
  return check_launch("kv_write");
}

template <typename XT>
static int launch_read(const ReadParams& p, int64_t count, int dw, cudaStream_t s) {
  const dim3 grid((unsigned)(count * (p.P / KV_TILE)), (unsigned)p.H, 2);
  if (dw == 64)       kv_read_kernel<XT, 64><<<grid, KW_THREADS, 0, s>>>(p);
  else if (dw == 128) kv_read_kernel<XT, 128><<<grid, KW_THREADS, 0, s>>>(p);
  else                kv_read_kernel<XT, 256><<<grid, KW_THREADS, 0, s>>>(p);
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
