// kv_plan.cu — block tables and slot maps of a paged K/V cache, on the GPU
// from the requests' lengths (wg_kv_plan).
//
// Request r holds L_r tokens after the step, n_r of them new. It has
// h_r = ceil((L_r - n_r) / page) pages and needs p_r = ceil(L_r / page); the
// p_r - h_r new ones come off the free list in request order. Slot of a token
// = its page * page size + its place in the page.
//
// Latency is what bounds it (a decode step plans a few hundred bytes), so the
// plan is one launch, and every CTA scans all requests itself (two integers a
// request) instead of waiting for another CTA's sums. Slots, the only output
// that can be long, are dealt over the CTAs' threads, four to a store, each
// found by a binary search in the tile's prefix sums. A cursor that is
// advanced in place must not be written before every CTA has read it: up to
// PLAN_CLUSTER CTAs are a cluster with a barrier for that, more leave the
// cursor to a second launch of one thread (1500 prompts of up to 448 tokens:
// 31 us with 8 CTAs, 13 to 17 with 64).
#include "ops.cuh"

namespace wg {
namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_CLUSTER = 8;
constexpr int PLAN_CTAS = 64;
constexpr int PLAN_MAX = 1 << 30;  // requests, and slots: the kernel steps 32-bit indices past them

struct PlanArgs {
  const int* lens;
  const int* fresh;
  int R, shift;
  const int* free_pages;
  int n_free;
  const int* cursor;
  int* cursor_out;
  int* table;
  int64_t ldt;
  int max_pages;
  int* slots;
  int n_slots;
  int* cu;
  int* status;
  bool barrier, advance;  // the CTAs are a cluster; this kernel writes the cursor
};

struct Two {
  long long a, b;
};
// Inclusive scan of (a, b) over the CTA; *total gets the sums.
__device__ Two block_scan(Two v, Two* total) {
  __shared__ Two warp_sum_sh[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) { v.a += a; v.b += b; }
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sum_sh[warp] = v;
  __syncthreads();
  Two w = warp_sum_sh[lane];  // 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o);
    if (lane >= o) { w.a += a; w.b += b; }
  }
  total->a = __shfl_sync(0xffffffffu, w.a, 31);
  total->b = __shfl_sync(0xffffffffu, w.b, 31);
  const long long pa = __shfl_sync(0xffffffffu, w.a, warp ? warp - 1 : 0);
  const long long pb = __shfl_sync(0xffffffffu, w.b, warp ? warp - 1 : 0);
  if (warp) { v.a += pa; v.b += pb; }
  return v;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}

// The cursor behind a plan whose CTAs could not be sure that all had read it.
__global__ void plan_cursor_kernel(const int* cursor, int* cursor_out, const int* status) {
  pdl_trigger();
  pdl_wait();
  *cursor_out = *cursor + status[1];
}

// grid (C, 1, 1), one cluster where p.barrier
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(PlanArgs p) {
  pdl_trigger();
  pdl_wait();
  const int rank = blockIdx.x, C = gridDim.x, tid = threadIdx.x;
  const int page = 1 << p.shift;
  const long long cursor = *p.cursor;
  // every length checked, and the sums that the whole step needs
  int code = 0;
  Two sum{0, 0};
  for (int r = tid; r < p.R; r += PLAN_THREADS) {
    const int L = p.lens[r], n = p.fresh[r];
    if (L < 0 || n < 0 || n > L) {
      code = max(code, WG_PLAN_BAD_LENGTH);
      continue;
    }
    const long long need = ((long long)L + page - 1) >> p.shift, held = ((long long)L - n + page - 1) >> p.shift;
    if (need > p.max_pages) code = max(code, WG_PLAN_TABLE_FULL);
    sum.a += n;
    sum.b += need - held;
  }
  Two total;
  block_scan(sum, &total);
  if (total.a > p.n_slots) code = max(code, WG_PLAN_SLOTS_FULL);
  if (cursor < 0 || cursor + total.b > p.n_free) code = max(code, WG_PLAN_NO_PAGES);
  __shared__ int code_sh;
  if (tid == 0) code_sh = 0;
  __syncthreads();
  if (code) atomicMax(&code_sh, code);
  __syncthreads();
  code = code_sh;
  if (p.barrier) cluster_sync();  // every CTA has read the cursor: it may be advanced in place
  else __syncthreads();           // (one CTA: every thread has)
  if (rank == 0 && tid == 0) {
    p.status[0] = code;
    p.status[1] = code ? 0 : (int)total.b;
    if (p.advance) *p.cursor_out = (int)(code ? cursor : cursor + total.b);
    p.cu[0] = 0;
  }
  const int live = code ? 0 : (int)total.a;
  for (int i = live + rank * PLAN_THREADS + tid; i < p.n_slots; i += C * PLAN_THREADS) p.slots[i] = -1;
  if (code) {
    for (int r = rank * PLAN_THREADS + tid; r < p.R; r += C * PLAN_THREADS) p.cu[r + 1] = 0;
    return;
  }
  // tiles of requests: prefix sums of new tokens and new pages
  __shared__ int end_sh[PLAN_THREADS];   // one past the request's last new token
  __shared__ int off_sh[PLAN_THREADS];   // its first new page's place in the free list
  __shared__ int held_sh[PLAN_THREADS];  // pages it holds already
  __shared__ int base_sh[PLAN_THREADS];  // tokens it held before
  Two carry{0, 0};
  const bool vec = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0;
  for (int r0 = 0; r0 < p.R; r0 += PLAN_THREADS) {
    const int r = r0 + tid, cnt = min(PLAN_THREADS, p.R - r0);
    Two v{0, 0};
    int L = 0, n = 0, held = 0;
    if (r < p.R) {
      L = p.lens[r];
      n = p.fresh[r];
      held = (int)(((long long)L - n + page - 1) >> p.shift);
      v.a = n;
      v.b = (((long long)L + page - 1) >> p.shift) - held;
    }
    const int extra = (int)v.b;
    v = block_scan(v, &total);
    const int first = (int)(carry.a), off = (int)(cursor + carry.b + v.b - extra);
    if (r < p.R) {
      end_sh[tid] = (int)(carry.a + v.a);
      off_sh[tid] = off;
      held_sh[tid] = held;
      base_sh[tid] = L - n;
      if (rank == tid % C) {
        p.cu[r + 1] = (int)(carry.a + v.a);
        int* row = p.table + (int64_t)r * p.ldt + held;
        for (int i = 0; i < extra; i++) row[i] = p.free_pages[off + i];
      }
    }
    __syncthreads();
    // the tile's tokens are [first, last); four consecutive ones per thread,
    // at multiples of four so that the store can be one vector
    const int last = end_sh[cnt - 1];
    for (int i0 = (first & ~3) + 4 * (rank * PLAN_THREADS + tid); i0 < last; i0 += 4 * C * PLAN_THREADS) {
      int lo = 0, hi = cnt - 1;  // first request whose end is past the token
      const int at = max(i0, first);
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end_sh[mid] > at) hi = mid;
        else lo = mid + 1;
      }
      int out[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = i0 + k;
        out[k] = -1;
        if (i < first || i >= last) continue;
        while (end_sh[lo] <= i) lo++;
        const int beg = lo ? end_sh[lo - 1] : first;
        const int pos = base_sh[lo] + (i - beg), col = pos >> p.shift;
        const int id = col < held_sh[lo] ? p.table[(int64_t)(r0 + lo) * p.ldt + col]
                                         : p.free_pages[off_sh[lo] + col - held_sh[lo]];
        // a page number that is none, or whose slots are past 32 bits, has none
        out[k] = id < 0 || id > (0x7fffffff >> p.shift) ? -1 : (id << p.shift) | (pos & (page - 1));
      }
      if (vec && i0 >= first && i0 + 4 <= last) {
        *reinterpret_cast<int4*>(p.slots + i0) = make_int4(out[0], out[1], out[2], out[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (i0 + k >= first && i0 + k < last) p.slots[i0 + k] = out[k];
      }
    }
    carry.a += total.a;
    carry.b += total.b;
    __syncthreads();  // the tile's arrays are free again
  }
}

}  // namespace
}  // namespace wg

extern "C" int wg_kv_plan(const int32_t* lens, const int32_t* new_tokens, int R, int page, const int32_t* free_pages,
                          int n_free, const int32_t* cursor, int32_t* cursor_out, int32_t* block_table,
                          int64_t ld_table, int max_pages, int32_t* slots, int n_slots, int32_t* cu_new,
                          int32_t* status, int device, void* stream) {
  using namespace wg;
  if (!lens || !new_tokens || !cursor || !cursor_out || !block_table || !cu_new || !status ||
      (n_free > 0 && !free_pages) || (n_slots > 0 && !slots)) {
    set_error("wg_kv_plan: null argument");
    return WG_ERR_INVALID;
  }
  if (!aligned4(lens, new_tokens, free_pages, cursor, cursor_out, block_table, slots, cu_new, status)) {
    set_error("wg_kv_plan: a tensor is not aligned to its type");
    return WG_ERR_INVALID;
  }
  if (R <= 0 || R > PLAN_MAX || !kv_page_ok(page) || n_free < 0 || n_slots < 0 || n_slots > PLAN_MAX || max_pages <= 0 ||
      ld_table < max_pages) {
    set_error("wg_kv_plan: bad argument (R %d and n_slots %d (at most %d), page %d (a power of two, 16 to 128), n_free %d, "
              "max_pages %d, ld_table %lld)", R, n_slots, PLAN_MAX, page, n_free, max_pages, (long long)ld_table);
    return WG_ERR_INVALID;
  }
  OpDevice dev;
  WG_CHECK(dev.enter("wg_kv_plan", device));
  // CTAs: four slots a thread, in a cluster while that suffices
  const int64_t work = (int64_t)n_slots + R;
  int C = 1;
  while (C < PLAN_CTAS && (int64_t)C * PLAN_THREADS * 4 < work) C *= 2;
  const bool cluster = C > 1 && C <= PLAN_CLUSTER, apart = C == 1 || cursor_out != cursor;
  PlanArgs a{lens, new_tokens, R, log2_of(page), free_pages, n_free, cursor, cursor_out, block_table, ld_table,
             max_pages, slots, n_slots, cu_new, status, cluster, cluster || apart};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(PLAN_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = cluster ? at : at + 1;
  cfg.numAttrs = (cluster ? 1 : 0) + (pdl_enabled() ? 1 : 0);
  WG_CHECK(launch_check(cudaLaunchKernelEx(&cfg, plan_kernel, a), "kv_plan"));
  if (a.advance) return WG_OK;
  return launch_check(launch_k(plan_cursor_kernel, dim3(1), dim3(1), 0, st, cursor, cursor_out, (const int*)status),
                      "kv_plan_cursor");
}
