// kv8.cu — the 8-bit paged K/V cache: writing tokens (wg_kv8_append) and
// reading them back (wg_kv8_read).
//
// A cached value is code * scale: int8 codes in [-127, 127], one fp32 scale
// for each (page, K or V, head). Scales are powers of two, the least 2^e
// (e >= -126) that takes the block's largest magnitude to at most 127 steps:
// x / scale, code * scale and the rescaling of a page that grows are then
// exact, so the only rounding is the one to the code (half to even) and a
// page that is filled token by token is rounded again only when its largest
// magnitude passes an octave, where amax / 127 would be rounded again with
// every new maximum. The price is a step of at most twice the finest one.
//
// Both are streams bounded by memory: K and V come in once (2 or 4 bytes a
// value) and go out as one byte, or the reverse.
#include "kernels.cuh"
#include "ops.cuh"

namespace wg {

int kv8_check(const char* what, const wg_kv8* c) {
  if (!c || !c->codes || !c->scales) {
    set_error("%s: null cache", what);
    return WG_ERR_INVALID;
  }
  if (c->num_pages <= 0 || c->n_kv_head <= 0 || !kv_page_ok(c->page) || (c->head_dim != 64 && c->head_dim != 128)) {
    set_error("%s: bad cache (%d pages of %d tokens (a power of two, 16 to 128), %d heads of %d (64 or 128))", what,
              c->num_pages, c->page, c->n_kv_head, c->head_dim);
    return WG_ERR_INVALID;
  }
  if ((int64_t)c->num_pages * c->page > 2147483647LL) {
    set_error("%s: %d pages of %d tokens need slots beyond 32 bits", what, c->num_pages, c->page);
    return WG_ERR_INVALID;
  }
  if (!aligned16(c->codes) || (reinterpret_cast<uintptr_t>(c->scales) & 3)) {
    set_error("%s: codes need 16-byte alignment, scales 4-byte", what);
    return WG_ERR_INVALID;
  }
  return WG_OK;
}

namespace {

// The power of two that takes amax to at most 127 steps; 0 for 0. amax =
// m * 2^k with m in [1, 2): 127 * 2^(k-6) = 1.984375 * 2^k holds it when
// m <= 1.984375, else 2^(k-5) does.
__device__ __forceinline__ float needed_scale(float amax) {
  if (!(amax > 0.f)) return 0.f;
  const uint32_t b = __float_as_uint(amax);
  const int k = (int)(b >> 23) - 127;  // subnormal amax: k = -127, clamped below
  int e = (b & 0x7fffffu) <= 0x7e0000u ? k - 6 : k - 5;
  e = max(e, -126);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// 8 consecutive elements as fp32.
__device__ __forceinline__ void load8(const void* p, int64_t i, int dt, bool vec, float (&x)[8]) {
  if (vec && dt == WG_DT_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i));
    const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else if (vec) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float2 f = dt_unpack2(dt, w[k]);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = dt_load(p, i + k, dt);
  }
}

__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  // NaN -> 0; an infinity (and what an infinity's neighbours cannot reach) -> +-127
  const float y = x * inv;
  const int c = y != y ? 0 : __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
  return (uint32_t)c & 255u;
}

struct AppendArgs {
  int8_t* codes;
  float* scales;
  int num_slots, shift, H, D;
  const void *k, *v;
  int64_t ldk, ldv;
  int dt;
  bool veck, vecv;
  const int* slots;
  int n, chunk, units;  // tokens, tokens per CTA, (K|V, head) pairs
};

constexpr int APPEND_WARPS = 8;
constexpr int APPEND_CHUNK = 64;  // most tokens a CTA looks for runs in

// One warp per (run of consecutive slots in a page, K or V, head). A CTA
// finds the runs that begin among its `chunk` tokens (grid x) and its warps
// deal the (run, unit) pairs of its 8 units (grid y).
__global__ void __launch_bounds__(APPEND_WARPS * 32) append_kernel(AppendArgs p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int start_sh[APPEND_CHUNK], len_sh[APPEND_CHUNK];
  __shared__ int runs_sh;
  const int t0 = blockIdx.x * p.chunk, tid = threadIdx.x;
  const int page = 1 << p.shift;
  if (tid == 0) runs_sh = 0;
  __syncthreads();
  if (tid < p.chunk && t0 + tid < p.n) {
    const int t = t0 + tid, s = p.slots[t];
    const int before = t ? p.slots[t - 1] : -1;
    if (s >= 0 && s < p.num_slots && (t == 0 || before != s - 1 || (s & (page - 1)) == 0)) {
      const int most = min(page - (s & (page - 1)), p.n - t);
      int len = 1;
      while (len < most && p.slots[t + len] == s + len) len++;
      const int k = atomicAdd(&runs_sh, 1);  // the order of the runs does not matter: each is written alone
      start_sh[k] = t;
      len_sh[k] = len;
    }
  }
  __syncthreads();
  const int runs = runs_sh, warp = tid >> 5, lane = tid & 31;
  const int u0 = blockIdx.y * APPEND_WARPS, nu = min(APPEND_WARPS, p.units - u0);
  const int per_tok = p.D >> 3;                 // lanes of 8 elements a token takes
  const int tok_step = 32 / per_tok;            // tokens a warp takes at once
  const int d = (lane % per_tok) * 8;
  for (int w = warp; w < runs * nu; w += APPEND_WARPS) {
    const int run = w / nu, unit = u0 + w % nu;  // unit = kv * H + head
    const int kv = unit >= p.H, head = unit - kv * p.H;
    const int t = start_sh[run], len = len_sh[run];
    const int slot = p.slots[t], id = slot >> p.shift, first = slot & (page - 1);
    const int64_t block = ((int64_t)id * 2 + kv) * p.H + head;
    int8_t* codes = p.codes + block * page * p.D;
    const float old = first ? p.scales[block] : 0.f;
    const void* src = kv ? p.v : p.k;
    const int64_t ld = kv ? p.ldv : p.ldk;
    const bool vec = kv ? p.vecv : p.veck;
    const int64_t col = (int64_t)head * p.D + d;
    float amax = 0.f;
    for (int i = lane / per_tok; i < len; i += tok_step) {
      float x[8];
      load8(src, (int64_t)(t + i) * ld + col, p.dt, vec, x);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float a = fabsf(x[k]);
        if (a <= 3.402823466e38f) amax = fmaxf(amax, a);  // finite values only
      }
    }
    amax = warp_max(amax);
    const float scale = fmaxf(old, needed_scale(amax));
    if (first && scale > old && old > 0.f) {
      // the page's earlier tokens in the new step: their codes are the only
      // copy, so they are rounded again (exact halving, half to even)
      const float ratio = old / scale;
      for (int i = lane * 8; i < first * p.D; i += 256) {
        uint2 v = *reinterpret_cast<uint2*>(codes + i);
        uint32_t in[2] = {v.x, v.y}, out[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int c = (int)(int8_t)(in[k >> 2] >> (8 * (k & 3)));
          out[k >> 2] |= ((uint32_t)__float2int_rn((float)c * ratio) & 255u) << (8 * (k & 3));
        }
        *reinterpret_cast<uint2*>(codes + i) = make_uint2(out[0], out[1]);
      }
    }
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    for (int i = lane / per_tok; i < len; i += tok_step) {
      float x[8];
      load8(src, (int64_t)(t + i) * ld + col, p.dt, vec, x);
      uint32_t out[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < 8; k++) out[k >> 2] |= code_of(x[k], inv) << (8 * (k & 3));
      *reinterpret_cast<uint2*>(codes + (int64_t)(first + i) * p.D + d) = make_uint2(out[0], out[1]);
    }
    if (lane == 0) p.scales[block] = scale;
  }
}

struct ReadArgs {
  const int8_t* codes;
  const float* scales;
  int num_slots, shift, H, D;
  void *k, *v;
  int64_t ldk, ldv;
  int dt;
  bool veck, vecv;
  const int* slots;
  int64_t total;  // n * 2 * H * D / 16
};

// One thread per 16 codes of (token, K or V, head).
__global__ void __launch_bounds__(256) read_kernel(ReadArgs p) {
  pdl_trigger();
  pdl_wait();
  const int per_head = p.D >> 4, per_tok = 2 * p.H * per_head;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.total; i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_tok), rest = (int)(i - (int64_t)t * per_tok);
    const int slot = p.slots[t];
    if (slot < 0 || slot >= p.num_slots) continue;  // no token: the row stays as it was
    const int unit = rest / per_head, d = (rest - unit * per_head) * 16;
    const int kv = unit >= p.H, head = unit - kv * p.H, page = 1 << p.shift;
    const int64_t block = ((int64_t)(slot >> p.shift) * 2 + kv) * p.H + head;
    const float scale = __ldg(p.scales + block);
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(p.codes + (block * page + (slot & (page - 1))) * p.D + d));
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; k++) x[k] = (float)(int)(int8_t)(w[k >> 2] >> (8 * (k & 3))) * scale;
    const int64_t at = (int64_t)t * (kv ? p.ldv : p.ldk) + (int64_t)head * p.D + d;
    void* dst = kv ? p.v : p.k;
    if (!(kv ? p.vecv : p.veck)) {
#pragma unroll
      for (int k = 0; k < 16; k++) dt_store(dst, at + k, p.dt, x[k]);
    } else if (p.dt == WG_DT_F32) {
      float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + at);
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
    } else {
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dst) + at);
#pragma unroll
      for (int k = 0; k < 2; k++)
        o[k] = make_uint4(dt_pack2(p.dt, x[8 * k], x[8 * k + 1]), dt_pack2(p.dt, x[8 * k + 2], x[8 * k + 3]),
                          dt_pack2(p.dt, x[8 * k + 4], x[8 * k + 5]), dt_pack2(p.dt, x[8 * k + 6], x[8 * k + 7]));
    }
  }
}

// Checks of a [n, heads, dim] tensor with rows of ld elements; *vec: whether
// every head of every row starts on 16 bytes.
int rows_check(const char* what, const char* name, const void* p, int dt, int64_t ld, int64_t width, bool* vec) {
  if (!p) {
    set_error("%s: %s is null", what, name);
    return WG_ERR_INVALID;
  }
  if (ld < width || ld > (int64_t)1 << 40) {
    set_error("%s: rows of %s are %lld elements apart, they hold %lld", what, name, (long long)ld, (long long)width);
    return WG_ERR_INVALID;
  }
  const int b = dt_bytes(dt);
  if (reinterpret_cast<uintptr_t>(p) % b) {
    set_error("%s: %s is not aligned to its type", what, name);
    return WG_ERR_INVALID;
  }
  *vec = aligned16(p) && ld * b % 16 == 0;
  return WG_OK;
}

}  // namespace

int launch_kv8_append(const wg_kv8& c, const void* k, const void* v, int dt, int64_t ldk, int64_t ldv, bool veck,
                      bool vecv, const int32_t* slots, int n, cudaStream_t st) {
  AppendArgs a{c.codes, c.scales, c.num_pages * c.page, log2_of(c.page), c.n_kv_head, c.head_dim, k, v, ldk, ldv,
               dt, veck, vecv, slots, n, 1, 2 * c.n_kv_head};
  // tokens a CTA looks through: few, so that short calls spread over the SMs
  // (every token may begin a run of its own), up to 64 where that leaves
  // enough CTAs
  const int gy = (a.units + APPEND_WARPS - 1) / APPEND_WARPS;
  while (a.chunk < APPEND_CHUNK && (int64_t)(n / (2 * a.chunk)) * gy >= 148 * 4) a.chunk *= 2;
  return launch_check(launch_k(append_kernel, dim3((n + a.chunk - 1) / a.chunk, gy), dim3(APPEND_WARPS * 32), 0, st, a),
                      "kv8_append");
}

}  // namespace wg

extern "C" int wg_kv8_append(const wg_kv8* cache, const void* k, const void* v, int dtype, int64_t ldk, int64_t ldv,
                             const int32_t* slots, int n, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_kv8_append";
  WG_CHECK(kv8_check(what, cache));
  if (!dt_ok(dtype) || n < 0 || (n > 0 && !slots)) {
    set_error("%s: bad argument (dtype %d, n %d)", what, dtype, n);
    return WG_ERR_INVALID;
  }
  if (n == 0) return WG_OK;
  bool vk, vv;
  const int64_t width = (int64_t)cache->n_kv_head * cache->head_dim;
  WG_CHECK(rows_check(what, "k", k, dtype, ldk, width, &vk));
  WG_CHECK(rows_check(what, "v", v, dtype, ldv, width, &vv));
  if (2 * cache->n_kv_head > 65535 * 8) {
    set_error("%s: too many heads", what);
    return WG_ERR_INVALID;
  }
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  return launch_kv8_append(*cache, k, v, dtype, ldk, ldv, vk, vv, slots, n, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int wg_kv8_read(const wg_kv8* cache, const int32_t* slots, int n, void* k, void* v, int dtype, int64_t ldk,
                           int64_t ldv, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_kv8_read";
  WG_CHECK(kv8_check(what, cache));
  if (!dt_ok(dtype) || n < 0 || (n > 0 && !slots)) {
    set_error("%s: bad argument (dtype %d, n %d)", what, dtype, n);
    return WG_ERR_INVALID;
  }
  if (n == 0) return WG_OK;
  bool vk, vv;
  const int64_t width = (int64_t)cache->n_kv_head * cache->head_dim;
  WG_CHECK(rows_check(what, "k", k, dtype, ldk, width, &vk));
  WG_CHECK(rows_check(what, "v", v, dtype, ldv, width, &vv));
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  ReadArgs a{cache->codes, cache->scales, cache->num_pages * cache->page, log2_of(cache->page), cache->n_kv_head,
             cache->head_dim, k, v, ldk, ldv, dtype, vk, vv, slots, (int64_t)n * 2 * width / 16};
  const int64_t blocks = (a.total + 255) / 256;
  return launch_check(launch_k(read_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(256), 0,
                               reinterpret_cast<cudaStream_t>(stream), a),
                      "kv8_read");
}
