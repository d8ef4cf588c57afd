// Packed-int4 matmul with a scale and a zero point per GROUP of the contraction axis and output channel:
//
//   w[k, n] = scale[k / g, n] * (code[k, n] - zero[k / g, n])
//   forward      out[m, n] = sum_k x[m, k] w[k, n]
//   transposed   out[m, k] = sum_n x[m, n] w[k, n]
//
// This file holds the dispatcher and the general kernel (any M, N, even K, pointers aligned to their element).  The decode
// kernel (w4_gemv.cu) and the kernel on CTA pairs (w4_pair.cu) take what fits them.
//
// General kernel: mma.sync with the weights as the 16-row operand, always as exact codes; what depends on the
// group is applied to fp32 numbers, so nothing but the sums is rounded:
//   forward      the sums of one group are finished with  total += scale * (sum - zero * sum_k x[m, k])  before the next
//                group's begin; the activations are summed up while they are staged;
//   transposed   scale varies along the contraction, the group along the rows: a tile's rows lie in one group, the
//                activations are multiplied with that group's scales while they are staged (products in fp32, split into
//                bf16 planes), and sum_n x scale zero is summed up beside it.
// Codes enter as code - 8 (exact): the sums and what the zero point takes off them are half as large.  The tensor core's
// sums truncate, so they are handed to fp32 totals at the latest every 128 indices (28672 in one chain: relative error 3.7e-5).
// 16-bit activations enter the forward product as they are; x * scale as two bf16 planes (16 bits of the product, below
// the result's own rounding); fp32 activations as three (all 24 bits).
// A long contraction with few tiles is split; the CTA that draws a tile's last ticket adds the slices in order.
//
// What is rounded is relative to scale |code - 8|: a weight of zero (code and zero point both 0, say) may bring 2^-14 of scale |x| (fp32:
// 2^-21) instead of nothing in the transposed product, whose planes hold x scale while the zero point's sum does not.
//
// Bound by the legacy tensor path and what feeds it (three planes of fp32 activations): 1024 x 4096 x 4096 fp32 502 us, 205
// TFLOP/s executed; transposed 553.  Small ones by latency: 137 x 272 x 909 fp32 13.5 us, transposed 14.8.
#include "w4_common.cuh"
#include "w4_plans.cuh"
#include <algorithm>
#include <cstring>

namespace jgq {

constexpr int WG_TOK = 64;                  // tokens per tile
constexpr int WG_KC = 32;                   // contraction indices per stage: a group is a multiple of it
constexpr int WG_THREADS = 128;
constexpr int WG_XSTRIDE = WG_KC + 8;       // elements per staged row: 80 bytes, eight rows start on eight different 16-byte banks

template <typename XT, bool TB> struct GroupType {                 // operand type and planes of the activations
  using CT = typename std::conditional<std::is_same<XT, __half>::value && !TB, __half, __nv_bfloat16>::type;
  static constexpr int PL = std::is_same<XT, float>::value ? 3 : (TB ? 2 : 1);
};

struct GroupParams {
  const void* x; const uint8_t* packed; const void* zero; const void* scale; void* out;
  float* part;                 // [splits][M][rows] when the contraction is split
  int32_t* tickets;            // one per tile of a split contraction, zero between launches
  int64_t M, N, K;
  int64_t rows, depth;         // weight rows of the product (N or K) and its contraction length (K or N)
  int group;
  int chunks_per_split, splits;
  int vec_w;                   // 4-byte loads of codes are legal
  int vec_x;                   // 16-byte loads of activations are legal
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// the low nibbles of the two halves, less 8
template <typename CT> __device__ __forceinline__ uint32_t centred(uint32_t v);
template <> __device__ __forceinline__ uint32_t centred<__half>(uint32_t v) {
  uint32_t r = (v & 0x000F000Fu) | 0x64006400u;
  const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__float2half_rn(1032.f)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t centred<__nv_bfloat16>(uint32_t v) {
  uint32_t r = (v & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&r), __float2bfloat162_rn(136.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename CT> __device__ __forceinline__ uint32_t pair_bits(float a, float b);
template <> __device__ __forceinline__ uint32_t pair_bits<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pair_bits<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// BM: weight rows per tile (32 or 64; in the transposed product a tile lies in one group)
template <typename XT, typename ZST, bool TB, int BM>
__global__ void __launch_bounds__(WG_THREADS)
w4_group_kernel(const GroupParams p) {
  using CT = typename GroupType<XT, TB>::CT;
  constexpr int PL = GroupType<XT, TB>::PL;
  constexpr int WM = BM / 32, WN = 4 / WM;             // warps along rows and tokens
  constexpr int NTW = WG_TOK / WN / 8;                 // token octets per warp
  constexpr int ASTRIDE = TB ? WG_KC + 8 : BM + 8;     // elements; forward: [contraction][row], transposed: [row][contraction]
  constexpr int AROWS = TB ? BM : WG_KC;
  constexpr int WORDS = BM * WG_KC / 8 / WG_THREADS;   // 4-byte words of codes per thread and stage
  __shared__ __align__(16) CT sa[2][AROWS * ASTRIDE];
  __shared__ __align__(16) CT sx[2][PL][WG_TOK * WG_XSTRIDE];
  __shared__ float scz[WG_TOK], sxs[2][WG_TOK];        // transposed: sum_n x scale zero; forward: a group's sums of x
  __shared__ int s_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int wm = (warp % WM) * 32, wn = (warp / WM) * (WG_TOK / WN);
  const int64_t row0 = (int64_t)blockIdx.x * BM, tok0 = (int64_t)blockIdx.y * WG_TOK;
  const int64_t chunks = (p.depth + WG_KC - 1) / WG_KC;
  const int64_t c_begin = (int64_t)blockIdx.z * p.chunks_per_split, c_end = min(chunks, c_begin + p.chunks_per_split);
  const int64_t tb_group = TB ? row0 / p.group : 0;

  // what a stage needs is requested a stage ahead (two ahead: 30 registers more, a CTA per SM less, up to 40 % slower)
  uint32_t wreg[WORDS];
  __align__(16) XT xraw[16];                        // as loaded: first touched when they are staged
  float s_lane = 0.f, z_lane = 0.f, cz = 0.f, xs = 0.f;
  ZST s_raw, z_raw;                                    // transposed: scale and zero point of index `lane` of the stage
  const int xt = tid >> 1, xh = (tid & 1) * 16;        // this thread's token of the tile and half of the stage's indices
  const XT* xrow = reinterpret_cast<const XT*>(p.x) + (tok0 + xt) * p.depth;
  const bool xlive = tok0 + xt < p.M;

  auto fetch = [&](int64_t c) {
    const int64_t d0 = c * WG_KC;
#pragma unroll
    for (int u = 0; u < WORDS; ++u) {
      const int i = tid + WG_THREADS * u;
      // forward: BM / 4 words of each of 16 byte rows; transposed: 8 words of each of BM / 2 byte rows
      const int64_t br = TB ? row0 / 2 + i / 8 : d0 / 2 + i / (BM / 4);
      const int64_t n = TB ? d0 + 4 * (i % 8) : row0 + 4 * (i % (BM / 4));
      uint32_t w = 0;
      if (2 * br < p.K && n < p.N) {
        const uint8_t* src = p.packed + br * p.N + n;
        if (p.vec_w) {
          w = *reinterpret_cast<const uint32_t*>(src);       // N % 4 == 0: the word is inside the row
        } else {                                             // out of the one or two aligned words that hold its bytes, others' bytes masked
          const uintptr_t at = reinterpret_cast<uintptr_t>(src);
          const uint32_t shift = 8 * (uint32_t)(at & 3), left = (uint32_t)min((int64_t)4, p.N - n);
          const uint32_t* lo = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
          const uint32_t w0 = lo[0], w1 = shift / 8 + left > 4 ? lo[1] : 0u;
          w = __funnelshift_r(w0, w1, shift) & (0xffffffffu >> (8 * (4 - left)));
        }
      }
      wreg[u] = w;
    }
    const int64_t d = d0 + xh;
    if (xlive && p.vec_x && d + 16 <= p.depth) {
#pragma unroll
      for (int v = 0; v < (int)sizeof(XT); ++v) reinterpret_cast<uint4*>(xraw)[v] = reinterpret_cast<const uint4*>(xrow + d)[v];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) xraw[i] = (xlive && d + i < p.depth) ? xrow[d + i] : from_f32<XT>(0.f);
    }
    if (TB) {
      const bool in = d0 + lane < p.depth;
      const int64_t o = tb_group * p.N + (in ? d0 + lane : 0);
      s_raw = in ? reinterpret_cast<const ZST*>(p.scale)[o] : from_f32<ZST>(0.f);
      z_raw = in ? reinterpret_cast<const ZST*>(p.zero)[o] : from_f32<ZST>(0.f);
    }
  };
  auto stage = [&](int buf, int64_t c) {
    CT* a = sa[buf];
    float xreg[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) xreg[i] = to_f32<XT>(xraw[i]);
    if (TB) {                                          // times this tile's scales; sum_n x scale zero beside it
      s_lane = to_f32<ZST>(s_raw);
      z_lane = to_f32<ZST>(z_raw) - 8.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        xreg[i] = __fmul_rn(xreg[i], __shfl_sync(0xffffffffu, s_lane, xh + i));
        cz = fmaf(xreg[i], __shfl_sync(0xffffffffu, z_lane, xh + i), cz);
      }
    }
    if (!TB) {
      float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 16; ++i) s4[i & 3] += xreg[i];
      xs += (s4[0] + s4[1]) + (s4[2] + s4[3]);
      if (c + 1 == c_end || (c + 1) * WG_KC % p.group == 0) {          // the group, or what of it lies in this slice, is complete
        xs += __shfl_xor_sync(0xffffffffu, xs, 1);
        if ((tid & 1) == 0) sxs[buf][xt] = xs;
        xs = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < WORDS; ++u) {
      const int i = tid + WG_THREADS * u;
      const uint32_t w = wreg[u];
      uint32_t e[2], o[2];                             // four channels of the even and of the odd contraction-axis index
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t b = __byte_perm(w, 0, h ? 0x4342 : 0x4140);       // two channels' bytes in the halves of a word
        e[h] = centred<CT>(b);
        o[h] = centred<CT>(b >> 4);
      }
      const int r = TB ? 2 * (i / 8) : 2 * (i / (BM / 4)), c = TB ? 4 * (i % 8) : 4 * (i % (BM / 4));
      *reinterpret_cast<uint2*>(a + r * ASTRIDE + c) = make_uint2(e[0], e[1]);
      *reinterpret_cast<uint2*>(a + (r + 1) * ASTRIDE + c) = make_uint2(o[0], o[1]);
    }
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
      uint32_t b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        b[i] = pair_bits<CT>(xreg[2 * i], xreg[2 * i + 1]);
        if (pl + 1 < PL) {                             // what this plane leaves; bf16 is the upper half of an fp32
          xreg[2 * i] -= __uint_as_float(b[i] << 16);
          xreg[2 * i + 1] -= __uint_as_float(b[i] & 0xffff0000u);
        }
      }
      uint4* dst = reinterpret_cast<uint4*>(&sx[buf][pl][xt * WG_XSTRIDE + xh]);
      dst[0] = make_uint4(b[0], b[1], b[2], b[3]);
      dst[1] = make_uint4(b[4], b[5], b[6], b[7]);
    }
  };

  float acc[2][NTW][4], total[2][NTW][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NTW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) { acc[i][j][e] = 0.f; total[i][j][e] = 0.f; }

  // The sums since the last call, all of one group (transposed: of any), into the totals.  Where the group ends, or the
  // slice, the zero point's part.
  auto hand_over = [&](int64_t grp, bool ends, int buf) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = row0 + wm + 16 * i + g + 8 * h;
        float s = 1.f, z = 0.f;
        if (!TB && n < p.rows) { s = zs_to_f32<ZST>(p.scale, grp * p.N + n); z = zs_to_f32<ZST>(p.zero, grp * p.N + n) - 8.f; }
#pragma unroll
        for (int j = 0; j < NTW; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = acc[i][j][2 * h + e];
            if (!TB && ends) v = fmaf(-z, sxs[buf][wn + 8 * j + 2 * q + e], v);
            total[i][j][2 * h + e] = TB ? total[i][j][2 * h + e] + v : fmaf(s, v, total[i][j][2 * h + e]);
            acc[i][j][2 * h + e] = 0.f;
          }
      }
  };

  if (c_begin < c_end) {
    fetch(c_begin);
    stage(0, c_begin);
  }
  __syncthreads();
  for (int64_t c = c_begin; c < c_end; ++c) {
    const int buf = (int)((c - c_begin) & 1);
    if (c + 1 < c_end) fetch(c + 1);
    const uint32_t ab = (uint32_t)__cvta_generic_to_shared(sa[buf]);
#pragma unroll
    for (int k16 = 0; k16 < WG_KC; k16 += 16) {
      uint32_t a[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (TB) ldsm_x4(a[i], ab + 2 * ((wm + 16 * i + (lane & 15)) * ASTRIDE + k16 + 8 * (lane >> 4)));
        else    ldsm_x4_t(a[i], ab + 2 * ((k16 + (lane & 7) + 8 * (lane >> 4)) * ASTRIDE + wm + 16 * i + 8 * ((lane >> 3) & 1)));
      }
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) {
        const uint32_t xb = (uint32_t)__cvta_generic_to_shared(sx[buf][pl]);
#pragma unroll
        for (int j = 0; j < NTW; j += 2) {
          uint32_t b[4];
          ldsm_x4(b, xb + 2 * ((wn + 8 * j + (lane & 7) + 8 * (lane >> 4)) * WG_XSTRIDE + k16 + 8 * ((lane >> 3) & 1)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            MmaType<CT>::mma(acc[i][j], a[i], b[0], b[1]);
            MmaType<CT>::mma(acc[i][j + 1], a[i], b[2], b[3]);
          }
        }
      }
    }
    {
      const int64_t k = (c + 1) * WG_KC;
      const bool ends = c + 1 == c_end || (!TB && k % p.group == 0);
      if (ends || k % 128 == 0) hand_over(TB ? 0 : c * WG_KC / p.group, ends, buf);
    }
    if (c + 1 < c_end) stage(buf ^ 1, c + 1);
    __syncthreads();
  }
  if (TB) {
    cz += __shfl_xor_sync(0xffffffffu, cz, 1);
    if ((tid & 1) == 0) scz[xt] = cz;
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < NTW; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = wn + 8 * j + 2 * q + e;
      const int64_t m = tok0 + t;
      if (m >= p.M) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t r = row0 + wm + 16 * i + g + 8 * h;
          if (r >= p.rows) continue;
          const float v = TB ? total[i][j][2 * h + e] - scz[t] : total[i][j][2 * h + e];
          if (p.splits > 1) p.part[((int64_t)blockIdx.z * p.M + m) * p.rows + r] = v;
          else reinterpret_cast<XT*>(p.out)[m * p.rows + r] = from_f32<XT>(v);
        }
    }
  if (p.splits > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      int32_t* ticket = p.tickets + blockIdx.y * gridDim.x + blockIdx.x;
      s_last = atomicAdd(ticket, 1) == p.splits - 1;
      if (s_last) *ticket = 0;                         // ready for the next launch
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const int rows = (int)min((int64_t)BM, p.rows - row0), toks = (int)min((int64_t)WG_TOK, p.M - tok0);
    const int64_t slice = p.M * p.rows;
    constexpr int E = 16;                              // elements of a thread whose slices are requested together
    for (int i0 = tid; i0 < toks * BM; i0 += E * WG_THREADS) {
      int64_t at[E];
      float sum[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e * WG_THREADS, t = i / BM, r = i % BM;
        at[e] = t < toks && r < rows ? (tok0 + t) * p.rows + row0 + r : -1;
        sum[e] = 0.f;
      }
      for (int z = 0; z < p.splits; ++z) {
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at[e] >= 0 ? __ldcg(p.part + z * slice + at[e]) : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += v[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at[e] >= 0) reinterpret_cast<XT*>(p.out)[at[e]] = from_f32<XT>(sum[e]);
    }
  }
}

// ------------------------------------------------------------------ host ----
// ---- which kernel ----
// Up to 32 rows, forward: the decode kernel (fp32 activations in passes of 16 rows).
constexpr int64_t kGroupDecodeRows = 32, kGroupPassRows = 16;
static bool group_decodes(int64_t M, int64_t N, int64_t K, int x_dtype, int transpose_b, int group) {
  return !transpose_b && M <= kGroupDecodeRows && plan_w4_gemv(x_dtype == JGQ_F32 ? std::min(M, kGroupPassRows) : M, N, K, x_dtype, group).use;
}
// 16-bit activations, more rows or transposed: CTA pairs.
static PairPlan group_pairs(int64_t M, int64_t N, int64_t K, int x_dtype, int transpose_b, int group) {
  return plan_w4_pair(M, N, K, x_dtype, transpose_b, group);
}

struct GroupPlan { int bm, tiles, mtiles, splits, chunks_per_split; size_t part_bytes; };

static GroupPlan plan_group(int64_t M, int64_t N, int64_t K, int group, int transpose_b) {
  GroupPlan pl;
  memset(&pl, 0, sizeof(pl));
  const int64_t rows = transpose_b ? K : N, depth = transpose_b ? N : K, chunks = cdiv(depth, WG_KC);
  pl.mtiles = (int)cdiv(M, WG_TOK);
  pl.bm = 64;
  // a transposed tile lies in one group; narrower tiles where the wide ones leave most SMs without one
  while (pl.bm > 32 && ((transpose_b && group % pl.bm != 0) || cdiv(rows, pl.bm) * pl.mtiles < sm_count() / 2)) pl.bm /= 2;
  pl.tiles = (int)cdiv(rows, pl.bm);
  // one resident wave of CTAs, of six stages at least
  const int64_t tiles = (int64_t)pl.tiles * pl.mtiles;
  const int64_t want = tiles > W4_TICKET_REGION / 4 ? 1 : std::max<int64_t>(1, 4 * (int64_t)sm_count() / tiles);
  const int64_t splits = std::min<int64_t>({want, cdiv(chunks, 6), 32});
  pl.chunks_per_split = (int)cdiv(chunks, splits);
  pl.splits = (int)cdiv(chunks, pl.chunks_per_split);
  pl.part_bytes = pl.splits > 1 ? align_up((size_t)pl.splits * M * rows * sizeof(float), 256) : 0;
  return pl;
}

template <typename XT, typename ZST, bool TB>
static int launch_group(const GroupPlan& pl, GroupParams& p, uint8_t* ws, cudaStream_t s) {
  p.part = reinterpret_cast<float*>(ws + W4_TICKET_REGION);
  p.tickets = reinterpret_cast<int32_t*>(ws);
  const dim3 grid((unsigned)pl.tiles, (unsigned)pl.mtiles, (unsigned)pl.splits);
  if (pl.bm == 64) w4_group_kernel<XT, ZST, TB, 64><<<grid, WG_THREADS, 0, s>>>(p);
  else             w4_group_kernel<XT, ZST, TB, 32><<<grid, WG_THREADS, 0, s>>>(p);
  return check_launch("w4_group_matmul");
}

}  // namespace jgq

using namespace jgq;

extern "C" size_t jgq_w4_group_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int group_size, int transpose_b) {
  if (M <= 0 || N <= 0 || K <= 0 || group_size <= 0) return 0;
  // over all activation types, and over the kernels that the alignment of the pointers chooses between
  const GroupPlan pl = plan_group(M, N, K, group_size, transpose_b);
  size_t bytes = W4_TICKET_REGION + pl.part_bytes;
  for (int dt : {JGQ_F32, JGQ_F16, JGQ_BF16}) {
    if (group_decodes(M, N, K, dt, transpose_b, group_size))
      for (int64_t rows : {M, std::min(M, kGroupPassRows), M % kGroupPassRows})
        for (int zb : {2, 4}) {
          const GemvPlan gp = plan_w4_gemv(rows, N, K, dt, group_size, zb);
          if (gp.use) bytes = std::max(bytes, gp.ws_bytes);
        }
    const PairPlan pp = group_pairs(M, N, K, dt, transpose_b, group_size);
    if (pp.use) bytes = std::max(bytes, pp.ws_bytes);
  }
  return bytes;
}

extern "C" int jgq_w4_group_matmul(const void* x, int x_dtype, const uint8_t* packed, const void* zero, const void* scale, int zs_dtype,
                                   void* out, int64_t M, int64_t N, int64_t K, int group_size, int flags,
                                   void* ws, size_t ws_bytes, void* stream) {
  JGQ_REQUIRE((flags & ~(JGQ_W4_TRANSPOSE_B | JGQ_W4_WEIGHTS_SETTLED)) == 0, JGQ_ERR_ARG, "w4_group_matmul: unknown flag bits %d", flags);
  const int transpose_b = flags & JGQ_W4_TRANSPOSE_B;
  JGQ_REQUIRE(x_dtype == JGQ_F32 || x_dtype == JGQ_F16 || x_dtype == JGQ_BF16, JGQ_ERR_ARG, "w4_group_matmul: activation dtype must be f32/f16/bf16");
  JGQ_REQUIRE(zs_dtype == JGQ_F32 || zs_dtype == JGQ_F16, JGQ_ERR_ARG, "w4_group_matmul: zero/scale dtype must be f32/f16");
  JGQ_REQUIRE(M >= 0 && N > 0 && K > 0, JGQ_ERR_ARG, "w4_group_matmul: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  JGQ_REQUIRE(K % 2 == 0, JGQ_ERR_ARG, "w4_group_matmul: K=%lld must be even (two codes per byte)", (long long)K);
  JGQ_REQUIRE(group_size > 0 && group_size % WG_KC == 0, JGQ_ERR_ARG, "w4_group_matmul: group_size %d is not a positive multiple of %d", group_size, WG_KC);
  // tokens: the grid's second dimension in tiles of 64
  JGQ_REQUIRE(M <= 65535ll * WG_TOK && N <= 2147483647LL / 4 && K <= 2147483647LL / 4, JGQ_ERR_LIMIT, "w4_group_matmul: shape too large");
  if (M == 0) return JGQ_OK;
  JGQ_REQUIRE(x && packed && zero && scale && out, JGQ_ERR_ARG, "w4_group_matmul: null pointer");
  const size_t zb = dtype_size(zs_dtype), xb = dtype_size(x_dtype);
  JGQ_REQUIRE(aligned(x, xb) && aligned(out, xb) && aligned(zero, zb) && aligned(scale, zb), JGQ_ERR_ALIGN, "w4_group_matmul: a pointer is not aligned to its element");
  // the kernel's own need: the entry point for it, which is asked once, covers every kernel and takes a microsecond
  auto fits = [&](size_t need) {
    return ws && ws_bytes >= need ? (int)JGQ_OK : fail(JGQ_ERR_WORKSPACE, "w4_group_matmul: workspace %zu < %zu bytes", ws_bytes, need);
  };
  int rc = fits(W4_TICKET_REGION);
  if (rc) return rc;
  JGQ_REQUIRE(aligned(ws, 256), JGQ_ERR_ALIGN, "w4_group_matmul: workspace must be 256-byte aligned");
  cudaStream_t s = (cudaStream_t)stream;
  const bool dense = aligned(packed, 16) && aligned(x, 16);
  const PairPlan pp = dense ? group_pairs(M, N, K, x_dtype, transpose_b, group_size) : PairPlan{};
  // 17 to 32 rows of 16 bits on large weights: on pairs that share the tiles (bf16, groups of 128, 17 and 32 rows: 4096 x 4096 20.7
  // and 20.8 us for 21.7 and 26.2; 8192 x 2048 22 for 23 and 28; 11008 x 4096 36.5 for 38 and 43; but 4096 x 2048 17.6 for 14.8 and 18.6)
  const bool paired = pp.use && M > 16 && K * N >= 1 << 24 && pp.splits > 1;
  if (!transpose_b && M <= kGroupDecodeRows && dense && !paired && aligned(out, x_dtype == JGQ_F32 ? 16 : 8) && aligned(scale, 16) && aligned(zero, 16)) {
    const int64_t step = x_dtype == JGQ_F32 ? std::min(M, kGroupPassRows) : M;
    const GemvPlan whole = plan_w4_gemv(step, N, K, x_dtype, group_size, (int)zb);
    if (whole.use) {
      const int64_t rest = M % step;                   // one pass, or two of fp32 activations
      const GemvPlan last = rest ? plan_w4_gemv(rest, N, K, x_dtype, group_size, (int)zb) : whole;
      rc = fits(std::max(whole.ws_bytes, last.ws_bytes));
      for (int64_t r0 = 0; r0 < M && !rc; r0 += step) {
        const int64_t rows = std::min(step, M - r0);
        rc = launch_w4_gemv(rows == step ? whole : last, (const char*)x + (size_t)r0 * K * xb, x_dtype, packed, zero, scale, zs_dtype,
                            (char*)out + (size_t)r0 * N * xb, rows, N, K, group_size, ws, (flags & JGQ_W4_WEIGHTS_SETTLED) != 0, s);
      }
      return rc;
    }
  }
  if (pp.use) {
    rc = fits(pp.ws_bytes);
    return rc ? rc : launch_w4_pair(pp, x, x_dtype, packed, zero, scale, zs_dtype, out, M, N, K, transpose_b, group_size, ws, s);
  }
  const GroupPlan pl = plan_group(M, N, K, group_size, transpose_b);
  rc = fits(W4_TICKET_REGION + pl.part_bytes);
  if (rc) return rc;
  GroupParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.packed = packed; p.zero = zero; p.scale = scale; p.out = out;
  p.M = M; p.N = N; p.K = K;
  p.rows = transpose_b ? K : N; p.depth = transpose_b ? N : K;
  p.group = group_size;
  p.chunks_per_split = pl.chunks_per_split; p.splits = pl.splits;
  p.vec_w = N % 4 == 0 && aligned(packed, 4);
  p.vec_x = p.depth * xb % 16 == 0 && aligned(x, 16);
  uint8_t* w = (uint8_t*)ws;
  const bool zf = zs_dtype == JGQ_F32;
#define JGQ_GROUP(XT)                                                                                                      \
  return transpose_b ? (zf ? launch_group<XT, float, true>(pl, p, w, s) : launch_group<XT, __half, true>(pl, p, w, s))       \
                     : (zf ? launch_group<XT, float, false>(pl, p, w, s) : launch_group<XT, __half, false>(pl, p, w, s))
  if (x_dtype == JGQ_F32) { JGQ_GROUP(float); }
  if (x_dtype == JGQ_F16) { JGQ_GROUP(__half); }
  JGQ_GROUP(__nv_bfloat16);
#undef JGQ_GROUP
}
