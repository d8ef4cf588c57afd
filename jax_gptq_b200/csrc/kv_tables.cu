// Block tables, slot maps and positions of a paged cache, from request lengths, on the device.
//
// State: block_table[B][W] (page of every block of P tokens; -1: none), held[B] (pages per request), a stack of free pages.
// One step, in this order:
//   finished requests give their pages back (pushed so that the first page of the first of them comes to lie on top);
//   every request gets the pages it lacks for lengths[r] + added[r] tokens, requests in order, popped from the stack;
//   slots / positions of the added tokens, cu_seqlens over the requests, lengths behind the step.
// All or nothing: if a request's tokens do not fit its row of the table, the stack has too few pages, more tokens are added than
// the slot map holds or a length is negative, no page is taken, every slot is -1, cu_seqlens is zero, lengths stay.  The first of these
// three is done by then: it does not depend on the rest, and doing it again does nothing.
//
// Latency-bound: one CTA of 1024 threads scans the requests (1024 at a time) twice, once for the totals; pages and, up to
// KT_SMALL of them, slots are handed out by all threads, each finding its request by bisection in the scanned sums.  Larger
// slot maps are filled by a second kernel over all SMs.  256 requests, one token each: 9 us; 1024 requests, some 300 000 tokens: 17 us.
#include "common.cuh"
#include <algorithm>
#include <cstring>

namespace jgq {

constexpr int KT_THREADS = 1024;
constexpr int KT_SMALL = 16384;            // slots that the first kernel fills itself

struct TableParams {
  int32_t* table; int32_t* held; int32_t* free_pages; int32_t* free_count;
  const int32_t* lengths; const int32_t* added; const uint8_t* finished;
  int64_t* slots; int32_t* positions; int32_t* cu; int32_t* lengths_out; int32_t* status;
  int64_t table_stride, max_tokens;
  int B, W, P, pages;
  int fill;                    // slots are filled here
};

// inclusive sums over the CTA of two values; `total` the CTA's
__device__ __forceinline__ void block_scan2(int64_t (&v)[2], int64_t (&total)[2], int64_t (*sw)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += u;
    }
  __syncthreads();
  if (lane == 31) { sw[warp][0] = v[0]; sw[warp][1] = v[1]; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int64_t w = sw[lane][i];
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    const int64_t before = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
    if (warp > 0) v[i] += before;
    total[i] = __shfl_sync(0xffffffffu, w, 31);
  }
}

// the i with before[i] <= x < before[i + 1]; before has n + 1 entries, before[0] <= x < before[n]
template <typename T>
__device__ __forceinline__ int bisect(const T* before, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)before[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(KT_THREADS) kv_tables_kernel(const TableParams p) {
  __shared__ int64_t sw[32][2];
  __shared__ int64_t s_pages[KT_THREADS + 1], s_tokens[KT_THREADS + 1];
  __shared__ int s_held[KT_THREADS], s_status;
  const int tid = threadIdx.x;
  int64_t count = min(max(0, *p.free_count), p.pages);
  if (tid == 0) s_status = 0;
  __syncthreads();

  // ---- pages of finished requests ----
  if (p.finished) {
    int64_t back = 0;
    for (int base = 0; base < p.B; base += KT_THREADS) {
      const int r = base + tid;
      int64_t v[2] = {r < p.B && p.finished[r] ? min(max(0, p.held[r]), p.W) : 0, 0}, total[2];
      block_scan2(v, total, sw);
      back += total[0];
    }
    if (back > p.pages - count) {                       // more than there are: the table was tampered with
      if (tid == 0) s_status = JGQ_KV_BAD_TABLE;
    } else if (back > 0) {
      int64_t at = 0;
      for (int base = 0; base < p.B; base += KT_THREADS) {
        const int r = base + tid;
        const int64_t mine = r < p.B && p.finished[r] ? min(max(0, p.held[r]), p.W) : 0;
        int64_t v[2] = {mine, 0}, total[2];
        block_scan2(v, total, sw);
        s_pages[tid + 1] = v[0];
        if (tid == 0) s_pages[0] = 0;
        __syncthreads();
        for (int64_t i = tid; i < total[0]; i += KT_THREADS) {
          const int w = bisect(s_pages, KT_THREADS, i);
          int32_t* e = p.table + (int64_t)(base + w) * p.table_stride + (i - s_pages[w]);
          p.free_pages[count + back - 1 - (at + i)] = *e;
          *e = -1;
        }
        if (mine > 0) p.held[r] = 0;
        at += total[0];
        __syncthreads();
      }
      count += back;
    }
  }
  __syncthreads();

  // ---- totals ----
  int64_t need = 0, tokens = 0;
  int bad = 0;
  for (int base = 0; base < p.B; base += KT_THREADS) {
    const int r = base + tid;
    int64_t v[2] = {0, 0}, total[2];
    if (r < p.B) {
      const int64_t len = p.lengths[r], add = p.added[r];
      if (len < 0 || add < 0 || len + add > 2147483647LL) bad |= JGQ_KV_BAD_LENGTH;
      const int64_t blocks = (max((int64_t)0, len + add) + p.P - 1) / p.P, held = p.held[r];
      if (blocks > p.W) bad |= JGQ_KV_ROW_FULL;
      if (held < 0 || held > p.W) bad |= JGQ_KV_BAD_TABLE;
      v[0] = max((int64_t)0, blocks - held);
      v[1] = max((int64_t)0, add);
    }
    block_scan2(v, total, sw);
    need += total[0];
    tokens += total[1];
  }
  if (need > count) bad |= JGQ_KV_NO_PAGES;
  if (tokens > p.max_tokens) bad |= JGQ_KV_TOO_MANY_TOKENS;
  if (bad) atomicOr(&s_status, bad);
  __syncthreads();
  const int status = s_status;
  if (tid == 0) {
    if (status) *p.status |= status;
    *p.free_count = (int32_t)(status ? count : count - need);
    p.cu[0] = 0;
  }

  // ---- hand out ----
  int64_t page_at = 0, token_at = 0;
  for (int base = 0; base < p.B; base += KT_THREADS) {
    const int r = base + tid;
    int64_t v[2] = {0, 0}, total[2];
    int held = 0, len = 0;
    if (r < p.B) {
      len = p.lengths[r];
      if (status) {
        p.cu[r + 1] = 0;
        p.lengths_out[r] = len;
      } else {
        const int add = p.added[r], blocks = (int)(((int64_t)len + add + p.P - 1) / p.P);
        held = p.held[r];
        v[0] = max(0, blocks - held);
        v[1] = add;
        p.held[r] = max(held, blocks);
        p.lengths_out[r] = len + add;
      }
    }
    if (status) continue;
    block_scan2(v, total, sw);
    s_pages[tid + 1] = v[0];
    s_tokens[tid + 1] = v[1];
    s_held[tid] = held;
    if (tid == 0) { s_pages[0] = 0; s_tokens[0] = 0; }
    if (r < p.B) p.cu[r + 1] = (int32_t)(token_at + v[1]);
    __syncthreads();
    for (int64_t i = tid; i < total[0]; i += KT_THREADS) {
      const int w = bisect(s_pages, KT_THREADS, i);
      p.table[(int64_t)(base + w) * p.table_stride + s_held[w] + (i - s_pages[w])] = p.free_pages[count - 1 - (page_at + i)];
    }
    __syncthreads();                                    // the pages are read below, by other threads
    if (p.fill) {
      for (int64_t i = tid; i < total[1]; i += KT_THREADS) {
        const int w = bisect(s_tokens, KT_THREADS, i);
        const int64_t pos = p.lengths[base + w] + (i - s_tokens[w]);
        p.slots[token_at + i] = (int64_t)p.table[(int64_t)(base + w) * p.table_stride + pos / p.P] * p.P + pos % p.P;
        p.positions[token_at + i] = (int32_t)pos;
      }
    }
    page_at += total[0];
    token_at += total[1];
    __syncthreads();
  }
  if (p.fill)
    for (int64_t i = (status ? 0 : tokens) + tid; i < p.max_tokens; i += KT_THREADS) { p.slots[i] = -1; p.positions[i] = 0; }
}

__global__ void __launch_bounds__(256) kv_slots_kernel(const TableParams p) {
  const int64_t tokens = p.cu[p.B];
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < p.max_tokens; i += gridDim.x * 256ll) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (i < tokens) {
      const int r = bisect(p.cu, p.B, i);
      pos = p.lengths[r] + (int32_t)(i - p.cu[r]);
      slot = (int64_t)p.table[(int64_t)r * p.table_stride + pos / p.P] * p.P + pos % p.P;
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
}

}  // namespace jgq

using namespace jgq;

extern "C" int jgq_kv_reserve(int32_t* block_table, int64_t table_stride, int64_t table_width, int32_t* held, int32_t* free_pages,
                              int32_t* free_count, int64_t pages, int page_size, const int32_t* lengths, const int32_t* added,
                              const uint8_t* finished, int64_t requests, int64_t* slots, int32_t* positions, int64_t max_tokens,
                              int32_t* cu_seqlens, int32_t* lengths_out, int32_t* status, void* stream) {
  JGQ_REQUIRE(requests >= 0 && table_width >= 0 && pages >= 1 && max_tokens >= 0, JGQ_ERR_ARG, "kv_reserve: bad sizes");
  JGQ_REQUIRE(page_size >= 1, JGQ_ERR_ARG, "kv_reserve: page_size %d", page_size);
  JGQ_REQUIRE(requests <= (1 << 20) && pages <= 2147483647LL && max_tokens <= (1 << 24) && table_width * page_size <= 2147483647LL, JGQ_ERR_LIMIT, "kv_reserve: shape too large");
  JGQ_REQUIRE((block_table || table_width == 0 || requests == 0) && free_pages && free_count && cu_seqlens && status, JGQ_ERR_ARG, "kv_reserve: null pointer");
  JGQ_REQUIRE(requests == 0 || (held && lengths && added && lengths_out), JGQ_ERR_ARG, "kv_reserve: null pointer");
  JGQ_REQUIRE(max_tokens == 0 || (slots && positions), JGQ_ERR_ARG, "kv_reserve: null pointer");
  JGQ_REQUIRE(lengths_out != lengths || requests == 0, JGQ_ERR_ARG, "kv_reserve: lengths_out must not be lengths");
  TableParams p;
  memset(&p, 0, sizeof(p));
  p.table = block_table; p.held = held; p.free_pages = free_pages; p.free_count = free_count;
  p.lengths = lengths; p.added = added; p.finished = finished;
  p.slots = slots; p.positions = positions; p.cu = cu_seqlens; p.lengths_out = lengths_out; p.status = status;
  p.table_stride = table_stride; p.max_tokens = max_tokens;
  p.B = (int)requests; p.W = (int)table_width; p.P = page_size; p.pages = (int)pages;
  p.fill = max_tokens <= KT_SMALL;
  cudaStream_t s = (cudaStream_t)stream;
  kv_tables_kernel<<<1, KT_THREADS, 0, s>>>(p);
  if (p.fill) return check_launch("kv_reserve");
  JGQ_LAUNCHED();
  kv_slots_kernel<<<(unsigned)std::min<int64_t>(cdiv(max_tokens, 256), 8 * (int64_t)sm_count()), 256, 0, s>>>(p);
  return check_launch("kv_reserve");
}
