// sample_rows.cu — drawing tokens with temperature, top-k, top-p and min-p
// from given random numbers (wg_sample_rows).
//
// With w_i = exp((x_i - max x) / T), every filter keeps a prefix of the row in
// descending order (lower index first among equals), so the kept set is one
// cut: the elements above a value, and the first J of those equal to it. Cuts
// are found without sorting, by a radix descent over the order-preserving bit
// patterns of the logits with a count and a mass for each digit.
//
// Which token a random number falls on is decided by sums of up to V weights,
// so the weights are evaluated in 64-bit floats and summed as integers in
// units of 2^-45 (at most 2^18 * 2^45 for a row): sums are exact and order
// free, and off by less than V * 2^-46 of the largest weight from the real
// ones.
#include "kernels.cuh"
#include "ops.cuh"

namespace wg {
namespace {

constexpr int SR_THREADS = 1024;
constexpr double SR_ONE = 35184372088832.0;  // 2^45
typedef unsigned long long u64;

struct Row {
  const void* p;
  int dt, V;
  __device__ __forceinline__ float at(int i) const {
    const float x = dt_load(p, i, dt);
    return x != x ? -INFINITY : x;
  }
};

// Unsigned keys in the order of the values (-0 with +0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

struct Weights {
  double zmax, t;
  float mx;
  __device__ __forceinline__ double operator()(float x) const { return x == mx ? 1.0 : exp((double)x / t - zmax); }
};
__device__ __forceinline__ u64 fixed_of(double w) { return __double2ull_rn(w * SR_ONE); }

__device__ u64 block_sum(u64 v) {
  __shared__ u64 part[32];
  __shared__ u64 total;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 s = 0;
    for (int w = 0; w < SR_THREADS / 32; w++) s += part[w];
    total = s;
  }
  __syncthreads();
  return total;
}

struct Cut {
  uint32_t key;  // elements above it are kept
  int ties;      // and so many of those equal to it, in index order
  u64 mass;      // their mass
};

// The shortest prefix of `in` (a cut itself) with at least k elements, or with
// a mass of at least `target` where by_mass.
__device__ Cut descend(const Row& row, const Weights& wt, const Cut& in, bool by_mass, u64 target) {
  __shared__ unsigned hc[256];
  __shared__ u64 hs[256];
  __shared__ uint32_t prefix_sh;
  __shared__ u64 above_sh, cabove_sh;
  __shared__ unsigned eq_sh;
  uint32_t prefix = 0, mask = 0;
  u64 above = 0, cabove = 0;  // mass and count of the elements above the current digits
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += SR_THREADS) { hc[i] = 0; hs[i] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < row.V; i += SR_THREADS) {
      const float x = row.at(i);
      const uint32_t key = key_of(x);
      if ((key & mask) != prefix || key <= in.key) continue;
      atomicAdd(&hc[(key >> shift) & 255], 1u);
      atomicAdd(&hs[(key >> shift) & 255], fixed_of(wt(x)));
    }
    if (threadIdx.x == 0 && (in.key & mask) == prefix && in.ties) {
      atomicAdd(&hc[(in.key >> shift) & 255], (unsigned)in.ties);
      atomicAdd(&hs[(in.key >> shift) & 255], (u64)in.ties * fixed_of(wt(of_key(in.key))));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int sel = -1, last = -1;
      u64 a = above, c = cabove;
      for (int d = 255; d >= 0; d--) {
        if (!hc[d]) continue;
        last = d;
        if ((by_mass ? a + hs[d] : c + hc[d]) >= target) { sel = d; break; }
        a += hs[d];
        c += hc[d];
      }
      if (sel < 0) {  // less than the target in all: everything is kept
        sel = last;
        a -= hs[sel];
        c -= hc[sel];
      }
      above_sh = a;
      cabove_sh = c;
      prefix_sh = prefix | ((uint32_t)sel << shift);
      eq_sh = hc[sel];
    }
    __syncthreads();
    above = above_sh;
    cabove = cabove_sh;
    prefix = prefix_sh;
    mask |= 255u << shift;
  }
  const u64 each = fixed_of(wt(of_key(prefix)));
  u64 j = by_mass ? (each ? (target > above ? (target - above + each - 1) / each : 1) : eq_sh)
                  : (target > cabove ? target - cabove : 1);
  if (j > eq_sh) j = eq_sh;
  if (j < 1) j = 1;
  __syncthreads();
  return Cut{prefix, (int)j, above + j * each};
}

struct Args {
  wg_sample s;
};

__global__ void __launch_bounds__(SR_THREADS) sample_rows_kernel(const Args a) {
  pdl_trigger();
  pdl_wait();
  const wg_sample& s = a.s;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row row{reinterpret_cast<const char*>(s.logits) + (int64_t)r * s.ld * dt_bytes(s.dtype), s.dtype, s.V};
  const float T = s.temperature ? s.temperature[r] : 1.f;
  const int k = s.top_k ? s.top_k[r] : 0;
  const float top_p = s.top_p ? s.top_p[r] : 1.f, min_p = s.min_p ? s.min_p[r] : 0.f;
  float u = s.u[r];
  if (!(u >= 0.f)) u = 0.f;
  // first maximum
  __shared__ u64 best_sh[32];
  u64 best = 0;
  for (int i = tid; i < s.V; i += SR_THREADS) {
    const u64 v = ((u64)key_of(row.at(i)) << 32) | (0xffffffffu - (uint32_t)i);
    best = v > best ? v : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if (lane == 0) best_sh[warp] = best;
  __syncthreads();
  best = best_sh[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  const float mx = of_key((uint32_t)(best >> 32));
  const int first = (int)(0xffffffffu - (uint32_t)best);
  if (mx == -INFINITY) {
    if (tid == 0) {
      s.tokens[r] = -1;
      if (s.logprobs) s.logprobs[r] = -INFINITY;
    }
    return;
  }
  const double t = T > 0.f ? (double)T : 1.0;
  const Weights wt{(double)mx / t, t, mx};
  u64 all = 0;
  for (int i = tid; i < s.V; i += SR_THREADS) all += fixed_of(wt(row.at(i)));
  all = block_sum(all);
  int token = first;
  if (T > 0.f) {
    Cut cut{0u, 0, all};  // everything (key 0 is no value's but -NaN's)
    if (k > 0 && k < s.V) cut = descend(row, wt, cut, false, (u64)k);
    if (!(top_p >= 1.f)) {
      const double goal = ceil((double)top_p * (double)cut.mass);
      cut = descend(row, wt, cut, true, goal >= 1.0 ? (u64)goal : 1);
    }
    // index of the last tie that is kept
    __shared__ int run_sh[SR_THREADS];
    __shared__ int last_sh, token_sh;
    const int per = (s.V + SR_THREADS - 1) / SR_THREADS, beg = min(s.V, tid * per), end = min(s.V, beg + per);
    int eq = 0;
    for (int i = beg; i < end; i++) eq += key_of(row.at(i)) == cut.key;
    run_sh[tid] = eq;
    if (tid == 0) last_sh = -1;
    __syncthreads();
    if (tid == 0) {
      int acc = 0;
      for (int w = 0; w < SR_THREADS; w++) { const int v = run_sh[w]; run_sh[w] = acc; acc += v; }
    }
    __syncthreads();
    if (eq && run_sh[tid] < cut.ties && cut.ties <= run_sh[tid] + eq) {
      int n = run_sh[tid];
      for (int i = beg; i < end; i++)
        if (key_of(row.at(i)) == cut.key && ++n == cut.ties) last_sh = i;
    }
    __syncthreads();
    const int last = last_sh;
    auto kept_mass = [&](int i) -> u64 {
      const float x = row.at(i);
      const uint32_t key = key_of(x);
      if (key < cut.key || (key == cut.key && i > last)) return 0;
      const double w = wt(x);
      return w >= (double)min_p || i == first ? fixed_of(w) : 0;
    };
    u64 mine = 0;
    for (int i = beg; i < end; i++) mine += kept_mass(i);
    const u64 mass = block_sum(mine);
    __shared__ u64 mass_sh[SR_THREADS];
    mass_sh[tid] = mine;
    if (tid == 0) token_sh = first;
    __syncthreads();
    if (tid == 0) {
      u64 acc = 0;
      for (int w = 0; w < SR_THREADS; w++) { const u64 v = mass_sh[w]; mass_sh[w] = acc; acc += v; }
    }
    __syncthreads();
    u64 goal = (u64)((double)u * (double)mass) + 1;
    if (goal > mass) goal = mass;
    u64 run = mass_sh[tid];
    if (run < goal && goal <= run + mine)
      for (int i = beg; i < end; i++) {
        run += kept_mass(i);
        if (run >= goal) {
          token_sh = i;
          break;
        }
      }
    __syncthreads();
    token = token_sh;
  }
  if (tid == 0) {
    s.tokens[r] = token;
    if (s.logprobs) {
      const float x = row.at(token);
      const double d = x == mx ? 0.0 : (double)x / t - wt.zmax;
      s.logprobs[r] = (float)(d - log((double)all / SR_ONE));
    }
  }
}

}  // namespace

int launch_sample_rows(const wg_sample& p, int device, cudaStream_t st) {
  (void)device;
  Args a{p};
  return launch_check(launch_k(sample_rows_kernel, dim3(p.R), dim3(SR_THREADS), 0, st, a), "sample_rows");
}

}  // namespace wg

extern "C" int wg_sample_rows(const wg_sample* p, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_sample_rows";
  if (!p || p->R < 0 || p->V <= 0 || p->V > (1 << 18) || p->ld < p->V) {
    set_error("%s: bad argument (V from 1 to %d, rows at least V apart)", what, 1 << 18);
    return WG_ERR_INVALID;
  }
  if (!dt_ok(p->dtype)) {
    set_error("%s: unsupported type %d", what, p->dtype);
    return WG_ERR_UNSUPPORTED;
  }
  if (p->R == 0) return WG_OK;
  if (!p->logits || !p->u || !p->tokens || reinterpret_cast<uintptr_t>(p->logits) % dt_bytes(p->dtype)) {
    set_error("%s: null or misaligned tensor", what);
    return WG_ERR_INVALID;
  }
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  return launch_sample_rows(*p, device, reinterpret_cast<cudaStream_t>(stream));
}
