// Packed-int4 forward matmul for a handful of token rows (M <= 32; 16 with fp32 activations): the decode kernel.
//
// HBM-bound: every packed byte is read once, by TMA, in 128-byte-row boxes (128 output channels
// wide, GV_ROWS byte rows deep) written with the 128-byte swizzle; each CTA keeps GV_NST boxes in
// flight and several CTAs share an SM.  The grid is one resident wave; the list of all stages,
// ordered by (channel group, contraction position), is cut into equal contiguous ranges, one per CTA.
//
// What the SM does per byte is kept small:
//   * a warp owns 32 channels of the box and walks every byte row of it, so that a channel's sum
//     over the CTA's contraction range lives in ONE warp: a flush is a few stores per warp, no
//     shared-memory reduction, no CTA-wide barrier.  Each warp draws its own ticket when slices of
//     several CTAs make up a channel group; the warp that draws the last one adds the slices in CTA
//     order (deterministic, no floating-point atomics) and writes the outputs;
//   * the weights are the 16-row operand of mma.sync m16n8k16.  A lane reads one 32-bit word (four
//     channels) from each of two consecutive byte rows; one byte permute per channel puts the two rows'
//     bytes of that channel into the two halves of a register, and two and-masks make two operand
//     registers of it: the low nibbles (contraction indices 2j, 2j+2) and the high nibbles (2j+1, 2j+3).
//     No exponent is or-ed in: a 4-bit code in the low mantissa bits of an f16 is the subnormal
//     code * 2^-24 (code * 2^-20 for the high nibble, where it sits four bits up), which the tensor
//     core multiplies exactly.  So an operand register costs 1.5 integer instructions;
//   * the activations are brought into that operand order once per stage and warp (shared memory,
//     a few hundred bytes): pairs (x[2j], x[2j+2]) and (x[2j+1], x[2j+3]), as they are.  An f16 MMA takes
//     the low nibbles of two steps, another their high nibbles into an accumulator of its own, which counts
//     a sixteenth: no activation is scaled, so none is rounded however small it is.  What an MMA reads of the
//     two steps lies side by side (even-index pairs of both, then in a second half the odd-index pairs), so that
//     one 8-byte load fills a register pair: with the pairs of a step side by side the moves cost up to 9 %;
//   * sum_k x[k], which the zero point multiplies, comes from one more MMA per step whose weight
//     operand is all ones.
// out[m, n] = scale[n] * (2^24 * acc[m, n] - zero[n] * sum_k x[m, k]).
//
// bf16 activations: a bf16 subnormal times an activation would leave fp32's range, so the codes get an exponent
// (0x4300 | code = 128 + code, the high nibbles shifted down first) and the 128 is taken off again on the FMA
// pipe: 2 logic operations and one subtraction per register instead of 1.5.  fp32 activations are two bf16 planes
// (x = hi + lo + O(2^-17 |x|)), two MMAs on the same expanded weights.
// More than eight token rows are groups of eight on the same expanded weights.
// Measured (GPU time per call, back to back): bf16 8 x 4096 x 11008 20.1 -> 18.0 us against the streaming kernel; f16 32 x 768 x
// 2304 28.5 -> 12.3 us against two passes of it.
//
// Scales per group of the contraction (FU > 0): a warp keeps the sums of the current group apart and, where the group ends,
// adds scale * (sum - zero * sum_k x) to totals, in fp32.  The scales and zero points of a stage's groups come by TMA with its
// box (requested one group ahead by each lane instead, 8192 x 28672 took 100 us with groups of 32; f16, one row, now: 36 us with groups
// of 128, 47 of 64, 55 of 32; 29 without groups).  FU is the number of 32-index units between two looks for a group's end: 4 where groups
// are multiples of 128, else 1.  A slice then holds the totals alone.  fp32 activations take three planes here (all 24
// bits), and codes other than f16's enter as code - 8, which halves what the zero point takes off again.
//
// Launch overlap: the kernel is launched with programmatic stream serialization.  It sets up its
// barriers and, when the caller declared the weights settled (JGQ_W4_WEIGHTS_SETTLED), issues its
// first boxes before `griddepcontrol.wait`, i.e. while the previous kernel on the stream is still
// finishing; activations, workspace and outputs are touched only after that wait.
#include "w4_common.cuh"
#include "w4_plans.cuh"
#include "umma.cuh"
#include "trace.cuh"
#include <algorithm>
#include <cstdlib>
#include <cstring>

// measurement builds: per CTA 0 entry, 1 past the grid-dependency wait, 2 first box landed, 3 last stage consumed, 4 exit
JGQ_TRACE_DEFINE(gemv, 8 * 1024)
#define GTRACE(i) JGQ_TRACE_CTA(gemv, i, 1024)

namespace jgq {

constexpr int GV_NST = 3;                      // boxes in flight per CTA
constexpr int GV_THREADS = WWARPS * 32;
constexpr int GV_MAX_SMEM = 200 * 1024;
constexpr int GV_TICKET_BYTES = W4_TICKET_REGION;   // one ticket per (channel group, warp): 1024 groups
__host__ __device__ constexpr int gemv_xs_tokens(int nt) { return nt > 16 ? nt : 16; }      // sum_k x slots per slice

struct GemvParams {
  const void* x; const void* zero; const void* scale; void* out;
  float* partials; int* tickets;
  int M, N, K;
  int ncg, spc;                // channel groups, stages per group
  int64_t S;                   // total stages
  int G;                       // CTAs
  int maxc;                    // slice slots per group
  int early;                   // 1: weights may be fetched before the stream's previous kernel has finished
  int group;                   // contraction indices per group
  int zs_bytes;                // of a scale or zero point (with groups; without, a template parameter says what they are)
  int zs_rows;                 // groups that a stage may touch
};

__device__ __forceinline__ int gemv_cta_of(int64_t idx, int64_t S, int G) {
  return (int)(((idx + 1) * G + S - 1) / S) - 1;     // the c with c*S/G <= idx < (c+1)*S/G
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(a) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// How an activation type enters the products.
template <typename XT> struct GemvType;
template <> struct GemvType<__half> {
  static constexpr int PLANES = 1;
  static constexpr int ACCS = 2;                                       // low and high nibbles apart
  static constexpr float UP = 16777216.f;                              // 2^24: the codes enter as code * 2^-24
  static constexpr uint32_t ONES = 0x3C003C00u;
  // four operand registers (low / high nibbles of two channels) of the two byte rows' permuted bytes
  template <bool CENTRED>
  __device__ static __forceinline__ void expand(uint32_t p0, uint32_t p1, uint32_t (&a)[4]) {
    a[0] = p0 & 0x000F000Fu; a[1] = p1 & 0x000F000Fu; a[2] = p0 & 0x00F000F0u; a[3] = p1 & 0x00F000F0u;
  }
  __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_f16(d, a0, a1, a2, a3, b0, b1);
  }
};
template <> struct GemvType<__nv_bfloat16> {
  static constexpr int PLANES = 1;
  static constexpr int ACCS = 1;
  static constexpr float UP = 1.f;
  static constexpr uint32_t ONES = 0x3F803F80u;
  template <bool CENTRED>
  __device__ static __forceinline__ uint32_t code(uint32_t v) {
    uint32_t r = (v & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&r), __float2bfloat162_rn(CENTRED ? 136.f : 128.f));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  template <bool CENTRED>
  __device__ static __forceinline__ void expand(uint32_t p0, uint32_t p1, uint32_t (&a)[4]) {
    a[0] = code<CENTRED>(p0); a[1] = code<CENTRED>(p1); a[2] = code<CENTRED>(p0 >> 4); a[3] = code<CENTRED>(p1 >> 4);
  }
  __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
  }
};
template <> struct GemvType<float> : GemvType<__nv_bfloat16> { static constexpr int PLANES = 2; };

__host__ __device__ constexpr int gemv_rows(int nt, int planes) { return nt * planes >= 32 ? 64 : 128; }      // byte rows per stage: the staged activations' registers
__host__ __device__ constexpr int gemv_ctas(int nt, int planes) { return nt * planes <= 2 ? 4 : (nt * planes <= 8 ? 3 : 2); }    // CTAs per SM the registers are capped for

// NT: token rows staged per warp (1, 2, 4, 8, 16 or 32 >= M); the MMA's n dimension holds eight of them, more
// rows are further such groups fed from the same expanded weights.  ROWS: byte rows per stage (64 or 128).
// FU: see above; 0: one scale per channel.
template <typename XT, int FU> __host__ __device__ constexpr int gemv_planes() { return std::is_same<XT, float>::value ? (FU ? 3 : 2) : 1; }
// bf16 activations of few rows, with groups: they enter as f16, like codes without conversion, after a power of two per row and stage
// that brings the largest to [2^13, 2^14) (what they say down to 2^-39 of it); a stage's sums are therefore finished with it.
// 8192 x 28672, groups of 128, one row: 48 -> 38 us, four rows 54 -> 48 (eight: no gain, every warp stages every row).
template <typename XT, int NT, int FU> __host__ __device__ constexpr bool gemv_scaled() { return FU > 0 && NT <= 4 && std::is_same<XT, __nv_bfloat16>::value; }
template <typename XT, int NT, typename ZST, int FU>
__global__ void __launch_bounds__(GV_THREADS, gemv_ctas(NT, gemv_planes<XT, FU>()))
w4_gemv_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap smap, const __grid_constant__ CUtensorMap zmap,
               const GemvParams p) {
  using namespace umma;
  constexpr bool SCALED = gemv_scaled<XT, NT, FU>();
  using T = GemvType<typename std::conditional<SCALED, __half, XT>::type>;
  constexpr int PL = gemv_planes<XT, FU>();
  constexpr bool GROUPED = FU > 0;
  constexpr bool CENTRED = GROUPED && !std::is_same<XT, __half>::value && !SCALED;
  constexpr int ROWS = gemv_rows(NT, PL);
  constexpr int STAGE_BYTES = ROWS * WCOLS;
  constexpr int STEPS = ROWS / 8;                  // 8 byte rows (16 contraction indices) per MMA step
  constexpr int PAIRS = ROWS / 2;                  // 8-byte operand pairs per token row and stage
  constexpr int XROW = PAIRS * 8 + 32;             // bytes per staged token row (+32: rows land on different banks)
  constexpr int XROW_ODD = PAIRS * 4;              // ACCS == 2: the odd-index pairs of a row
  constexpr int XWARP = NT * PL * XROW;            // planes one after the other
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* zs_ring = ring + GV_NST * STAGE_BYTES;  // with groups: per stage scales [zs_rows][128], then zero points
  const int zs_half = GROUPED ? p.zs_rows * WCOLS * p.zs_bytes : 0;
  uint8_t* xs_all = zs_ring + GV_NST * 2 * zs_half;   // [warp][token row][PAIRS] operand pairs, then one row of zeros
  __shared__ __align__(8) uint64_t full_bar[GV_NST];
  __shared__ int issued[GV_NST];
  __shared__ int done[GV_NST];
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int64_t idx_begin = ((int64_t)blockIdx.x * p.S) / p.G;
  const int64_t idx_end = ((int64_t)(blockIdx.x + 1) * p.S) / p.G;
  const int nstage = (int)(idx_end - idx_begin);
  const int g_begin = (int)(idx_begin / p.spc);
  const int st_begin = (int)(idx_begin - (int64_t)g_begin * p.spc);
  volatile int* abort_flag = &s_abort;

  auto issue_stage = [&](int j) {
    const int lin = st_begin + j;
    const int gg = g_begin + lin / p.spc, ss = lin % p.spc;
    const int slot = j % GV_NST;
    issued[slot] = j;
    mbar_expect_tx(&full_bar[slot], STAGE_BYTES + 2 * zs_half);
    tma_load_2d(ring + slot * STAGE_BYTES, &wmap, gg * WCOLS, ss * ROWS, &full_bar[slot]);
    if (GROUPED) {
      const int row = ss * (2 * ROWS) / p.group;
      tma_load_2d(zs_ring + slot * 2 * zs_half, &smap, gg * WCOLS, row, &full_bar[slot]);
      tma_load_2d(zs_ring + slot * 2 * zs_half + zs_half, &zmap, gg * WCOLS, row, &full_bar[slot]);
    }
  };

  GTRACE(0);
  if (threadIdx.x == 0) {
    for (int i = 0; i < GV_NST; ++i) { mbar_init(&full_bar[i], 1); done[i] = 0; issued[i] = -1; }
    s_abort = 0;
    fence_barrier_init();
    prefetch_tensormap(&wmap);
    if (GROUPED) { prefetch_tensormap(&smap); prefetch_tensormap(&zmap); }
  }
  // the row of zeros that lanes of absent token rows read
  for (int i = threadIdx.x; i < XROW / 4; i += GV_THREADS)
    reinterpret_cast<uint32_t*>(xs_all + WWARPS * XWARP)[i] = 0u;
  __syncthreads();
  if (p.early && threadIdx.x == 0)
    for (int j = 0; j < GV_NST && j < nstage; ++j) issue_stage(j);
  // Wait until everything enqueued before this kernel has completed: activations, workspace and outputs
  // are only touched below this line.  Only then is the next kernel on the stream allowed to begin its
  // own set-up: whatever it reads early was therefore complete before THIS kernel's predecessor ended.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  GTRACE(1);
  if (!p.early && threadIdx.x == 0)
    for (int j = 0; j < GV_NST && j < nstage; ++j) issue_stage(j);

  constexpr int NG = (NT + 7) / 8;               // groups of eight token rows
  constexpr int ACCS = T::ACCS;
  float acc[NG][2][ACCS][4], accx[NG][4];
  auto clear_acc = [&]() {
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        accx[q][i] = 0.f;
#pragma unroll
        for (int h = 0; h < ACCS; ++h) { acc[q][0][h][i] = 0.f; acc[q][1][h][i] = 0.f; }
      }
  };
  clear_acc();
  // with groups: totals of this lane's channels and tokens
  float tot[GROUPED ? NG : 1][2][4];
  auto clear_tot = [&]() {
#pragma unroll
    for (int q = 0; q < (GROUPED ? NG : 1); ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) { tot[q][0][i] = 0.f; tot[q][1][i] = 0.f; }
  };
  clear_tot();
  float down[SCALED ? NT : 1];                   // what takes the power of two of a stage's activations off again, per row
  // the sums since the last call, which belong to the group in row `row` of stage `slot`'s scales, into the totals
  auto finish_group = [&](int slot, int row) {
    float sc[4], z[4];
    const uint8_t* at = zs_ring + slot * 2 * zs_half + (row * WCOLS + 32 * warp + 4 * g) * p.zs_bytes;
    if (p.zs_bytes == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(at), v = *reinterpret_cast<const uint2*>(at + zs_half);
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
      const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), d = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
      sc[0] = a.x; sc[1] = a.y; sc[2] = b.x; sc[3] = b.y;
      z[0] = c.x; z[1] = c.y; z[2] = d.x; z[3] = d.y;
    } else {
      const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + zs_half);
      sc[0] = a.x; sc[1] = a.y; sc[2] = a.z; sc[3] = a.w;
      z[0] = b.x; z[1] = b.y; z[2] = b.z; z[3] = b.w;
    }
#pragma unroll
    for (int q = 0; q < (GROUPED ? NG : 1); ++q)
#pragma unroll
      for (int tile = 0; tile < 2; ++tile)
#pragma unroll
        for (int i = 0; i < 4; ++i) {                  // channel 2 tile + i / 2 of the four, token 2 t + i % 2
          if (NT == 1 && (i & 1)) continue;            // one token row: column 0 alone
          const int c = 2 * tile + (i >> 1);
          const float v = ACCS == 2 ? fmaf(acc[q][tile][ACCS - 1][i], 0.0625f, acc[q][tile][0][i]) : acc[q][tile][0][i];
          float sum = fmaf(-(CENTRED ? z[c] - 8.f : z[c]), accx[q][i & 1], v * T::UP);
          if constexpr (SCALED) sum *= NT == 1 ? down[0] : NT == 2 ? down[i & 1] : t == 0 ? down[i & 1] : down[NT == 4 ? 2 + (i & 1) : 0];
          tot[q][tile][i] = fmaf(sc[c], sum, tot[q][tile][i]);
        }
    clear_acc();
  };

  const uint32_t ring_u32 = smem_u32(ring);
  const uint32_t xs_warp = smem_u32(xs_all) + warp * XWARP;
  // this lane's operand pairs: token row g (+ 8 in the second group) when present, else the row of zeros
  uint32_t xs_read[NG];
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int row = g + 8 * q;
    xs_read[q] = (row < p.M && row < NT ? xs_warp + row * XROW : smem_u32(xs_all) + WWARPS * XWARP) + t * 8;
  }
  // byte rows 8*sl + 2t and + 1 of a step, 32-bit word of channels 32*warp + 4g .. + 3; the 16-byte chunk
  // index is xor-ed with (row & 7) by the swizzle, and row & 7 does not depend on the step
  const uint32_t chunk = 2 * warp + (g >> 2), inchunk = 4 * (g & 3);
  const uint32_t off0 = (2 * t) * WCOLS + ((chunk ^ (2 * t)) << 4) + inchunk;
  const uint32_t off1 = (2 * t + 1) * WCOLS + ((chunk ^ (2 * t + 1)) << 4) + inchunk;
  constexpr uint32_t ones = T::ONES;

  int gid = g_begin, st = st_begin;
  int group_now = GROUPED ? st * (2 * ROWS) / p.group : 0, group_end = GROUPED ? (group_now + 1) * p.group : 0;      // current group, and the index behind it
  bool alive = true;
  for (int s = 0; s < nstage; ++s) {
    const int cg = gid;
    const int slot = s % GV_NST;
    // ---- activations of this stage: four values per token row and load, issued before the wait ----
    constexpr bool kF32 = std::is_same<XT, float>::value;
    using XV = typename std::conditional<kF32, float4, uint2>::type;
    XV xv[NT][ROWS / 64];
    {
      const int k0 = st * (2 * ROWS);
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int h = 0; h < ROWS / 64; ++h) {
          const int k = k0 + 4 * (lane + 32 * h);
          xv[r][h] = XV{};
          // Not through the read-only path: the previous kernel may write them while this one is already running.
          if (r < p.M && k < p.K)        // K % 8 == 0: the four values are inside the row together
            xv[r][h] = *reinterpret_cast<const XV*>((const XT*)p.x + (int64_t)r * p.K + k);
        }
    }
    if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&full_bar[slot], (s / GV_NST) & 1, abort_flag));
    if (s == 0) GTRACE(2);
    __syncwarp();                          // the previous stage's operand pairs have been read by every lane
    float up = 1.f;
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int h = 0; h < ROWS / 64; ++h) {
        // operand order: (x[k], x[k+2]) and (x[k+1], x[k+3])
        const uint32_t dst = xs_warp + r * XROW + (lane + 32 * h) * 8;
        if constexpr (kF32) {
          const float f[4] = {xv[r][h].x, xv[r][h].z, xv[r][h].y, xv[r][h].w};
          uint32_t hi[2], lo[2], least[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const __nv_bfloat16 h0 = __float2bfloat16_rn(f[2 * i]), h1 = __float2bfloat16_rn(f[2 * i + 1]);
            const float r0 = f[2 * i] - __bfloat162float(h0), r1 = f[2 * i + 1] - __bfloat162float(h1);
            const __nv_bfloat16 l0 = __float2bfloat16_rn(r0), l1 = __float2bfloat16_rn(r1);
            hi[i] = (uint32_t)__bfloat16_as_ushort(h0) | ((uint32_t)__bfloat16_as_ushort(h1) << 16);
            lo[i] = (uint32_t)__bfloat16_as_ushort(l0) | ((uint32_t)__bfloat16_as_ushort(l1) << 16);
            if (PL == 3) {
              const __nv_bfloat16 m0 = __float2bfloat16_rn(r0 - __bfloat162float(l0)), m1 = __float2bfloat16_rn(r1 - __bfloat162float(l1));
              least[i] = (uint32_t)__bfloat16_as_ushort(m0) | ((uint32_t)__bfloat16_as_ushort(m1) << 16);
            }
          }
          sts64(dst, hi[0], hi[1]);
          sts64(dst + NT * XROW, lo[0], lo[1]);
          if (PL == 3) sts64(dst + 2 * NT * XROW, least[0], least[1]);
        } else {
          uint32_t ev, od;
          if constexpr (SCALED) {
            if (h == 0) {
              uint32_t top = 0;
#pragma unroll
              for (int j = 0; j < ROWS / 64; ++j) top = __vmaxu2(top, __vmaxu2(xv[r][j].x & 0x7fff7fffu, xv[r][j].y & 0x7fff7fffu));
              const uint32_t e = min(max(__reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16)) >> 7, 14u), 254u);
              up = __uint_as_float((267u - e) << 23);
              down[r] = __uint_as_float((e - 13u) << 23);
            }
            const __half2 a = __floats2half2_rn(__uint_as_float(xv[r][h].x << 16) * up, __uint_as_float(xv[r][h].y << 16) * up);
            const __half2 b = __floats2half2_rn(__uint_as_float(xv[r][h].x & 0xffff0000u) * up, __uint_as_float(xv[r][h].y & 0xffff0000u) * up);
            ev = *reinterpret_cast<const uint32_t*>(&a);
            od = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            ev = __byte_perm(xv[r][h].x, xv[r][h].y, 0x5410);
            od = __byte_perm(xv[r][h].x, xv[r][h].y, 0x7632);
          }
          if constexpr (ACCS == 2) {
            // pair `lane & 3` of step lane / 4: 8 bytes per pair for two steps
            const uint32_t dst2 = xs_warp + r * XROW + h * 128 + (lane >> 3) * 32 + (lane & 3) * 8 + ((lane >> 2) & 1) * 4;
            sts32(dst2, ev);
            sts32(dst2 + XROW_ODD, od);
          } else {
            sts64(dst, ev, od);
          }
        }
      }
    __syncwarp();
    if (alive) {
      const uint32_t tile = ring_u32 + slot * STAGE_BYTES;
      auto words = [&](uint32_t (&w)[ACCS][2], int sl) {       // of ACCS steps of 16 contraction indices
#pragma unroll
        for (int h = 0; h < ACCS; ++h) {
          w[h][0] = lds32(tile + (sl + h) * (8 * WCOLS) + off0);
          w[h][1] = lds32(tile + (sl + h) * (8 * WCOLS) + off1);
        }
      };
      auto steps = [&](const uint32_t (&w)[ACCS][2], int sl) {
        uint32_t a0[ACCS][4], a1[ACCS][4];         // per step: low nibbles, then high nibbles, of the two channel tiles
#pragma unroll
        for (int h = 0; h < ACCS; ++h) {
          const uint32_t w1 = w[h][0], w2 = w[h][1];
          T::template expand<CENTRED>(__byte_perm(w1, w2, 0x4400), __byte_perm(w1, w2, 0x5511), a0[h]);
          T::template expand<CENTRED>(__byte_perm(w1, w2, 0x6622), __byte_perm(w1, w2, 0x7733), a1[h]);
        }
#pragma unroll
        for (int q = 0; q < NG; ++q)
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) {
            const uint32_t xr = xs_read[q] + pl * (q * 8 + g < p.M ? NT * XROW : 0) + sl * (32 / ACCS);
            const uint2 xb = lds64(xr);
            if constexpr (ACCS == 2) {
              const uint2 xc = lds64(xr + XROW_ODD);
              T::mma(acc[q][0][0], a0[0][0], a0[0][1], a0[1][0], a0[1][1], xb.x, xb.y);
              T::mma(acc[q][1][0], a1[0][0], a1[0][1], a1[1][0], a1[1][1], xb.x, xb.y);
              T::mma(accx[q], ones, ones, ones, ones, xb.x, xb.y);
              T::mma(acc[q][0][1], a0[0][2], a0[0][3], a0[1][2], a0[1][3], xc.x, xc.y);
              T::mma(acc[q][1][1], a1[0][2], a1[0][3], a1[1][2], a1[1][3], xc.x, xc.y);
              T::mma(accx[q], ones, ones, ones, ones, xc.x, xc.y);
            } else {
              T::mma(acc[q][0][0], a0[0][0], a0[0][1], a0[0][2], a0[0][3], xb.x, xb.y);
              T::mma(acc[q][1][0], a1[0][0], a1[0][1], a1[0][2], a1[0][3], xb.x, xb.y);
              T::mma(accx[q], ones, ones, ones, ones, xb.x, xb.y);
            }
          }
      };
      if constexpr (!GROUPED) {
#pragma unroll
        for (int sl = 0; sl < STEPS; sl += ACCS) {
          uint32_t w[ACCS][2];
          words(w, sl);
          steps(w, sl);
        }
      } else {
        int k = st * (2 * ROWS);
        const int first = k / p.group;                 // the stage's row 0 of scales
        bool pending = false;
        // the words of the next CB steps are read before the products of these
        constexpr int CB = FU >= 2 ? 4 : 2, CN = CB / ACCS;
        uint32_t w[2][CN][ACCS][2];
        auto chunk_words = [&](uint32_t (&c)[CN][ACCS][2], int sl) {
#pragma unroll
          for (int i = 0; i < CN; ++i) words(c[i], sl + i * ACCS);
        };
        auto chunk_steps = [&](const uint32_t (&c)[CN][ACCS][2], int sl) {
#pragma unroll
          for (int i = 0; i < CN; ++i) steps(c[i], sl + i * ACCS);
        };
        chunk_words(w[0], 0);
#pragma unroll 1
        for (int s0 = 0; s0 < STEPS; s0 += 2 * FU) {
          if constexpr (2 * FU == 2 * CB) {
            chunk_words(w[1], s0 + CB);
            chunk_steps(w[0], s0);
            if (s0 + 2 * CB < STEPS) chunk_words(w[0], s0 + 2 * CB);
            chunk_steps(w[1], s0 + CB);
          } else {
            static_assert(2 * FU == CB, "a look for the group's end per chunk, or per two");
            if (s0 + CB < STEPS) chunk_words(w[1], s0 + CB);
            chunk_steps(w[0], s0);
#pragma unroll
            for (int i = 0; i < CN; ++i)
#pragma unroll
              for (int h = 0; h < ACCS; ++h) { w[0][i][h][0] = w[1][i][h][0]; w[0][i][h][1] = w[1][i][h][1]; }
          }
          k += 32 * FU;
          pending = k != group_end;
          if (!pending) {
            finish_group(slot, group_now - first);
            ++group_now;
            group_end += p.group;
          }
        }
        // the channel group's last stage, or this CTA's: what its last group has so far
        if (pending && (SCALED || st == p.spc - 1 || s == nstage - 1)) finish_group(slot, group_now - first);
      }
      __syncwarp();
      if (lane == 0) {
        int old;
        asm volatile("atom.acq_rel.cta.shared.add.u32 %0, [%1], 1;" : "=r"(old) : "r"(smem_u32(&done[slot])) : "memory");
        if (old == WWARPS - 1) {               // every warp has read the slot: refill it
          done[slot] = 0;
          if (s + GV_NST < nstage) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            issue_stage(s + GV_NST);
          }
        }
      }
    }
    const int st_now = st;
    st = (st + 1 == p.spc) ? 0 : st + 1;
    if (st == 0) ++gid;
    const bool last_of_group = (st_now == p.spc - 1) || (s == nstage - 1);
    if (!last_of_group) continue;
    if (s == nstage - 1) GTRACE(3);

    // ---- flush this warp's 32 channels of group cg ----
    // lane (g, t): tokens 2t and 2t+1; channels n0 .. n0+3 = (tile 0 row g, tile 0 row g+8, tile 1 row g, tile 1 row g+8)
    const float kUp = GROUPED ? 1.f : T::UP;
    const int n0 = cg * WCOLS + 32 * warp + 4 * g;
    const int first_c = gemv_cta_of((int64_t)cg * p.spc, p.S, p.G);
    const int last_c = gemv_cta_of((int64_t)(cg + 1) * p.spc - 1, p.S, p.G);
    const int ncontrib = last_c - first_c + 1;
    const float poison = (alive && !*abort_flag) ? 0.f : __int_as_float(0x7fc00000);
    float4 v[NG][2];
    float xsum[NG][2];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        auto sum = [&](int tile, int i) {
          if constexpr (GROUPED) return tot[q][tile][i] + poison;
          else if constexpr (ACCS == 2) return fmaf(acc[q][tile][1][i], 0.0625f, acc[q][tile][0][i]) + poison;
          else return acc[q][tile][0][i] + poison;
        };
        v[q][e] = make_float4(sum(0, e), sum(0, 2 + e), sum(1, e), sum(1, 2 + e));
        xsum[q][e] = accx[q][e];
      }
    bool write_out = true;
    if (ncontrib > 1) {
      constexpr int SL = NT * 32 + gemv_xs_tokens(NT);        // floats per (slot, warp): NT token rows x 32 channels, then sum_k x
      float* base = p.partials + ((int64_t)cg * p.maxc * WWARPS + warp) * SL;
      float* mine = base + (int64_t)(blockIdx.x - first_c) * WWARPS * SL;
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = 8 * q + 2 * t + e;
          if (tok < p.M && tok < NT) {
            *reinterpret_cast<float4*>(mine + tok * 32 + 4 * g) = v[q][e];
            if (!GROUPED && g == 0) mine[NT * 32 + tok] = xsum[q][e];
          }
        }
      __threadfence();
      __syncwarp();
      int last = 0;
      if (lane == 0) {
        const int old = atomicAdd(&p.tickets[cg * WWARPS + warp], 1);
        last = (old == ncontrib - 1);
        if (last) p.tickets[cg * WWARPS + warp] = 0;           // ready for the next launch
      }
      last = __shfl_sync(0xffffffffu, last, 0);
      write_out = last != 0;
      if (write_out) {
        __threadfence();
#pragma unroll
        for (int q = 0; q < NG; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = 8 * q + 2 * t + e;
            v[q][e] = make_float4(0.f, 0.f, 0.f, 0.f);
            xsum[q][e] = 0.f;
            if (tok < p.M && tok < NT) {
              for (int zc = 0; zc < ncontrib; ++zc) {            // slices are added in CTA order: deterministic
                const float* src = base + (int64_t)zc * WWARPS * SL;
                const float4 a = __ldcg(reinterpret_cast<const float4*>(src + tok * 32 + 4 * g));
                v[q][e].x += a.x; v[q][e].y += a.y; v[q][e].z += a.z; v[q][e].w += a.w;
                if (!GROUPED) xsum[q][e] += __ldcg(src + NT * 32 + tok);
              }
            }
          }
      }
    }
    if (write_out && n0 < p.N) {               // N % 16 == 0: the four channels are inside together
      float sc[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { sc[i] = 1.f; z[i] = 0.f; if (!GROUPED) { sc[i] = zs_to_f32<ZST>(p.scale, n0 + i); z[i] = zs_to_f32<ZST>(p.zero, n0 + i); } }
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = 8 * q + 2 * t + e;
          if (tok < p.M && tok < NT) {
            const float o0 = GROUPED ? v[q][e].x : sc[0] * (kUp * v[q][e].x - z[0] * xsum[q][e]), o1 = GROUPED ? v[q][e].y : sc[1] * (kUp * v[q][e].y - z[1] * xsum[q][e]);
            const float o2 = GROUPED ? v[q][e].z : sc[2] * (kUp * v[q][e].z - z[2] * xsum[q][e]), o3 = GROUPED ? v[q][e].w : sc[3] * (kUp * v[q][e].w - z[3] * xsum[q][e]);
            XT* dst = (XT*)p.out + (int64_t)tok * p.N + n0;
            if constexpr (kF32) {
              *reinterpret_cast<float4*>(dst) = make_float4(o0, o1, o2, o3);
            } else {
              const XT o[4] = {from_f32<XT>(o0), from_f32<XT>(o1), from_f32<XT>(o2), from_f32<XT>(o3)};
              *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
            }
          }
        }
    }
    clear_acc();
    if (GROUPED) {                                   // the next channel group begins at contraction index 0
      clear_tot();
      group_now = 0;
      group_end = p.group;
    }
  }

  GTRACE(4);
  // After a timed-out wait some boxes may still be in flight: give them a bounded time to land before
  // the CTA's shared memory is released.
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) {
    for (int i = 0; i < GV_NST; ++i) {
      const int j = issued[i];
      if (j < 0) continue;
      const long long t0 = clock64();
      while (!mbar_try_wait(&full_bar[i], (j / GV_NST) & 1) && clock64() - t0 < 20000000LL) {}
    }
  }
}

// ------------------------------------------------------------------ host ----

// groups of scales that a stage of `span` contraction indices may touch
static int gemv_zs_rows(int span, int group) { return group % span == 0 ? 1 : span % group == 0 ? span / group : span / group + 2; }

GemvPlan plan_w4_gemv(int64_t M, int64_t N, int64_t K, int x_dtype, int group, int zs_bytes) {
  GemvPlan pl;
  memset(&pl, 0, sizeof(pl));
  const int planes = x_dtype == JGQ_F32 ? (group ? 3 : 2) : 1;
  if (M < 1 || M > (planes > 1 ? 16 : 32) || N % 16 != 0 || K % 8 != 0) return pl;
  pl.ncg = (int)cdiv(N, WCOLS);
  if (pl.ncg * WWARPS > GV_TICKET_BYTES / (int)sizeof(int)) return pl;
  pl.use = 1;
  pl.nt = M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : M <= 8 ? 8 : M <= 16 ? 16 : 32;
  pl.rows = gemv_rows(pl.nt, planes);
  pl.spc = (int)cdiv(K / 2, pl.rows);
  pl.S = (int64_t)pl.ncg * pl.spc;
  const int xrow = (pl.rows / 2) * 8 + 32;
  pl.zs_rows = group ? gemv_zs_rows(2 * pl.rows, group) : 0;
  pl.smem_bytes = GV_NST * (pl.rows * WCOLS + 2 * pl.zs_rows * WCOLS * zs_bytes) + 1024 + (WWARPS * pl.nt * planes + 1) * xrow;
  const int by_smem = (227 * 1024) / (pl.smem_bytes + 1024 + 128);
  const int per_sm = std::max(1, std::min(gemv_ctas(pl.nt, planes), by_smem));
  pl.G = (int)std::min<int64_t>(per_sm * (int64_t)sm_count(), std::max<int64_t>(1, pl.S / 2));   // one resident wave
  const int64_t per = pl.S / pl.G;                    // every CTA streams per or per + 1 stages
  pl.maxc = (int)cdiv(pl.spc, per) + 1;
  pl.part_bytes = align_up((size_t)pl.ncg * pl.maxc * WWARPS * (pl.nt * 32 + gemv_xs_tokens(pl.nt)) * sizeof(float), 256);
  pl.ws_bytes = GV_TICKET_BYTES + pl.part_bytes;
  return pl;
}

template <typename XT, int NT, typename ZST, int FU>
static int launch_gemv_inst(const GemvPlan& pl, const GemvParams& p, const CUtensorMap& wmap, const CUtensorMap& smap, const CUtensorMap& zmap, cudaStream_t s) {
  auto kern = w4_gemv_kernel<XT, NT, ZST, FU>;
  struct AttrTag {};
  const int arc = once_per_device<AttrTag>([&]() {         // with groups the size varies: as much as any call may want
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FU ? GV_MAX_SMEM : pl.smem_bytes);
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);   // a hint: all of it as shared memory
    cudaGetLastError();
    return (int)e;
  });
  if (arc != 0) return fail(JGQ_ERR_CUDA, "w4_matmul: cannot raise the dynamic shared memory limit");
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)pl.G);
  cfg.blockDim = dim3(GV_THREADS);
  cfg.dynamicSmemBytes = (size_t)pl.smem_bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, wmap, smap, zmap, p);
  note_launches(1);
  if (e != cudaSuccess) { cudaGetLastError(); return fail(JGQ_ERR_CUDA, "w4_gemv: %s", cudaGetErrorString(e)); }
  return JGQ_OK;
}

template <typename XT, typename ZST, int FU>
static int launch_gemv_type(const GemvPlan& pl, const GemvParams& p, const CUtensorMap& wmap, const CUtensorMap& smap, const CUtensorMap& zmap, cudaStream_t s) {
  switch (pl.nt) {
    case 1:  return launch_gemv_inst<XT, 1, ZST, FU>(pl, p, wmap, smap, zmap, s);
    case 2:  return launch_gemv_inst<XT, 2, ZST, FU>(pl, p, wmap, smap, zmap, s);
    case 4:  return launch_gemv_inst<XT, 4, ZST, FU>(pl, p, wmap, smap, zmap, s);
    case 8:  return launch_gemv_inst<XT, 8, ZST, FU>(pl, p, wmap, smap, zmap, s);
    case 16: return launch_gemv_inst<XT, 16, ZST, FU>(pl, p, wmap, smap, zmap, s);
    default:
      if constexpr (GemvType<XT>::PLANES == 1) return launch_gemv_inst<XT, 32, ZST, FU>(pl, p, wmap, smap, zmap, s);
      return fail(JGQ_ERR_ARG, "w4_gemv: bad plan");
  }
}

int launch_w4_gemv(const GemvPlan& pl, const void* x, int x_dtype, const uint8_t* packed, const void* zero, const void* scale,
                   int zs_dtype, void* out, int64_t M, int64_t N, int64_t K, int group, void* ws, int settled, cudaStream_t s) {
  CUtensorMap wmap;
  const int rc = encode_tmap_2d_u8(&wmap, packed, (uint64_t)N, (uint64_t)(K / 2), (uint64_t)N, WCOLS, (uint32_t)pl.rows, 1);
  if (rc) return rc;
  GemvParams p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.zero = zero; p.scale = scale; p.out = out;
  p.tickets = (int*)ws;
  p.partials = (float*)((char*)ws + GV_TICKET_BYTES);
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.ncg = pl.ncg; p.spc = pl.spc; p.S = pl.S; p.G = pl.G; p.maxc = pl.maxc;
  p.early = settled ? 1 : 0;
  if (group > 0) {
    p.group = group;
    p.zs_bytes = dtype_size(zs_dtype);
    p.zs_rows = pl.zs_rows;
    CUtensorMap smap, zmap;
    const uint64_t groups = (uint64_t)cdiv(K, group);
    int zrc = encode_tmap_2d_zs(&smap, scale, zs_dtype, (uint64_t)N, groups, WCOLS, (uint32_t)pl.zs_rows);
    if (!zrc) zrc = encode_tmap_2d_zs(&zmap, zero, zs_dtype, (uint64_t)N, groups, WCOLS, (uint32_t)pl.zs_rows);
    if (zrc) return zrc;
#define JGQ_GEMV(XT) return group % 128 == 0 ? launch_gemv_type<XT, float, 4>(pl, p, wmap, smap, zmap, s) : launch_gemv_type<XT, float, 1>(pl, p, wmap, smap, zmap, s)
    if (x_dtype == JGQ_F16) { JGQ_GEMV(__half); }
    if (x_dtype == JGQ_BF16) { JGQ_GEMV(__nv_bfloat16); }
    JGQ_GEMV(float);
#undef JGQ_GEMV
  }
  const CUtensorMap &smap = wmap, &zmap = wmap;            // not used
  const bool zf = zs_dtype == JGQ_F32;
  if (x_dtype == JGQ_F16) return zf ? launch_gemv_type<__half, float, 0>(pl, p, wmap, smap, zmap, s) : launch_gemv_type<__half, __half, 0>(pl, p, wmap, smap, zmap, s);
  if (x_dtype == JGQ_BF16)
    return zf ? launch_gemv_type<__nv_bfloat16, float, 0>(pl, p, wmap, smap, zmap, s) : launch_gemv_type<__nv_bfloat16, __half, 0>(pl, p, wmap, smap, zmap, s);
  return zf ? launch_gemv_type<float, float, 0>(pl, p, wmap, smap, zmap, s) : launch_gemv_type<float, __half, 0>(pl, p, wmap, smap, zmap, s);
}

}  // namespace jgq
