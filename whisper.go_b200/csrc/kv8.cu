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
// Both are streams bounded by memory: K and V come in (2 or 4 bytes a value;
// once where a run of tokens in a page holds up to 8 KB a head, which a warp
// keeps while it looks for the largest magnitude: 64 tokens of 64 16-bit values;
// of longer runs all but the last 8 KB are read a second time) and go out as one
// byte, or the reverse. Measured on 96000 tokens of 20 heads of 64 in f16 in
// pages of 64 (737 MB each way): append 150 us = 4.9 TB/s, 75 % of the measured
// copy rate (16 warps an SM); read 137 us = 5.4 TB/s, 82 %. Small calls (64
// tokens) are launches and the host's part, 6.5 to 9 us each.
#include "kernels.cuh"
#include "ops.cuh"

namespace wg {

int kv8_check(const char* what, const wg_kv8* c) {
  if (!c || !c->codes || !c->scales) {
    set_error("%s: null cache", what);
    return WG_ERR_INVALID;
  }
  if (c->num_pages <= 0 || c->n_kv_head <= 0 || c->n_kv_head > 65536 || !kv_page_ok(c->page) || (c->head_dim != 64 && c->head_dim != 128)) {
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

// 16 bytes of a row: 8 elements of 16 bits or 4 of 32.
template <int ES>
__device__ __forceinline__ uint4 load16(const void* p, int64_t i, bool vec) {
  const uint8_t* at = reinterpret_cast<const uint8_t*>(p) + i * ES;
  if (vec) return __ldg(reinterpret_cast<const uint4*>(at));
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if (ES == 4) w[k] = __ldg(reinterpret_cast<const uint32_t*>(at) + k);
    else
      w[k] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + 2 * k) |
             (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + 2 * k + 1) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Their values.
template <int ES>
__device__ __forceinline__ void values16(uint4 v, int dt, float (&x)[16 / ES]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if constexpr (ES == 4) {
      x[k] = __uint_as_float(w[k]);
    } else {
      const float2 f = dt_unpack2(dt, w[k]);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}

// Codes of 4 values as bytes. x / scale is exact (a power of two), so the one
// rounding is that of the sum with 1.5 * 2^23, whose low byte is the nearest
// integer, half to even. Finite values need no clamp: |x| <= 127 * scale.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  const float magic = 12582912.f;
  const uint32_t lo = __byte_perm(__float_as_uint(fmaf(a, inv, magic)), __float_as_uint(fmaf(b, inv, magic)), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(fmaf(c, inv, magic)), __float_as_uint(fmaf(d, inv, magic)), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// NaN as 0, an infinity as 127 steps.
__device__ __forceinline__ float tame(float x, float scale) {
  const float most = 127.f * scale;
  return x != x ? 0.f : fminf(fmaxf(x, -most), most);
}
// Largest magnitude in 16 bytes, as the bits of its type (what is not finite is
// larger than anything finite), joined into m: two 16-bit maxima, or one of 32.
template <int ES>
__device__ __forceinline__ uint32_t join_max(uint32_t m, uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; k++) m = ES == 2 ? __vmaxu2(m, w[k] & 0x7fff7fffu) : max(m, w[k] & 0x7fffffffu);
  return m;
}

struct AppendArgs {
  int8_t* codes;
  float* scales;
  int num_slots, shift, H, D;
  const void *k, *v;
  int64_t ldk, ldv;
  int64_t head_step, batch_step;  // elements between heads, and between batches of `batch` tokens
  int batch;
  int dt;
  bool veck, vecv;
  const int* slots;
  int n, chunk, units, group;  // tokens, tokens per CTA, (K|V, head) pairs, pairs per CTA
};

constexpr int APPEND_WARPS = 8;
constexpr int APPEND_CHUNK = 64;  // most tokens a CTA looks for runs in
constexpr int APPEND_HOLD = 16;   // 16-byte pieces a lane holds between the two passes over a run
constexpr int PAGE_MAX = 128;

// One warp per (run of consecutive slots in a page, K or V, head). A CTA
// finds the runs that begin among its `chunk` tokens (grid x) and its warps
// deal the (run, unit) pairs of its 8 units (grid y). The run's values stay in
// registers between finding the largest magnitude and coding (8 KB a warp: a
// page of 64 tokens of 64 16-bit values), so they are read once; of what is
// longer the last block is held and the ones before it are read again.
template <int ES>
__global__ void __launch_bounds__(APPEND_WARPS * 32) append_kernel(AppendArgs p) {
  pdl_trigger();
  pdl_wait();
  constexpr int EPL = 16 / ES;  // elements a lane takes at once
  __shared__ int slot_sh[APPEND_CHUNK + PAGE_MAX + 1];
  __shared__ uint32_t begin_sh[(APPEND_CHUNK + PAGE_MAX) / 32 + 1];  // bit i: a run begins at token t0 + i, or none goes on
  __shared__ short start_sh[APPEND_CHUNK], len_sh[APPEND_CHUNK];
  __shared__ int runs_sh;
  const int t0 = blockIdx.x * p.chunk, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int page = 1 << p.shift, look = p.chunk + page;  // a run that begins in the chunk ends within `look`
  // tokens before and after the rows count as outside
  if (tid <= look) {
    const int t = t0 + tid - 1;
    slot_sh[tid] = t >= 0 && t < p.n ? p.slots[t] : -1;
  }
  if (tid == 0) runs_sh = 0;
  __syncthreads();
  {
    bool begins = true;
    if (tid < look) {
      const int s = slot_sh[tid + 1];
      begins = s < 0 || s >= p.num_slots || slot_sh[tid] != s - 1 || (s & (page - 1)) == 0;
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, begins);
    if (lane == 0 && warp <= look / 32) begin_sh[warp] = bits;
  }
  __syncthreads();
  if (tid < p.chunk) {
    const int s = slot_sh[tid + 1];
    if ((begin_sh[tid >> 5] >> (tid & 31) & 1) && s >= 0 && s < p.num_slots) {
      int w = (tid + 1) >> 5;  // the next beginning is the end
      uint32_t rest = begin_sh[w] >> ((tid + 1) & 31) << ((tid + 1) & 31);
      while (!rest && (w + 1) * 32 <= look) rest = begin_sh[++w];
      const int end = rest ? min(look, w * 32 + __ffs(rest) - 1) : look;
      const int k = atomicAdd(&runs_sh, 1);  // the order of the runs does not matter: each is written alone
      start_sh[k] = (short)tid;
      len_sh[k] = (short)min(end - tid, page - (s & (page - 1)));
    }
  }
  __syncthreads();
  const int runs = runs_sh;
  const int u0 = blockIdx.y * p.group, nu = min(p.group, p.units - u0);
  const int per_tok = p.D / EPL;         // lanes that a token takes
  const int tok_step = 32 / per_tok;     // tokens a warp takes at once
  const int sub = lane / per_tok, d = (lane % per_tok) * EPL;
  const int block_len = APPEND_HOLD * tok_step;
  for (int w = warp; w < runs * nu; w += APPEND_WARPS) {
    const int run = w / nu, unit = u0 + w % nu;  // unit = kv * H + head
    const int kv = unit >= p.H, head = unit - kv * p.H;
    const int len = len_sh[run], slot = slot_sh[start_sh[run] + 1];
    const int id = slot >> p.shift, first = slot & (page - 1);
    const int64_t block = ((int64_t)id * 2 + kv) * p.H + head;
    int8_t* codes = p.codes + block * page * p.D;
    const float old = first ? p.scales[block] : 0.f;
    const void* src = kv ? p.v : p.k;
    const int64_t ld = kv ? p.ldv : p.ldk;
    const bool vec = kv ? p.vecv : p.veck;
    // a run lies in one batch: batches begin pages of their own
    const int t_run = t0 + start_sh[run], in_batch = t_run / p.batch;
    const int64_t from = in_batch * p.batch_step + (int64_t)(t_run - in_batch * p.batch + sub) * ld + head * p.head_step + d;
    uint4 raw[APPEND_HOLD];
    auto load = [&](int b0) {
#pragma unroll
      for (int i = 0; i < APPEND_HOLD; i++) {
        const int tok = b0 + i * tok_step;
        raw[i] = tok + sub < len ? load16<ES>(src, from + tok * ld, vec) : make_uint4(0, 0, 0, 0);
      }
    };
    uint32_t bits = 0;
    int held = 0;
    for (int b0 = 0; b0 < len; b0 += block_len) {
      load(b0);
      held = b0;
#pragma unroll
      for (int i = 0; i < APPEND_HOLD; i++) bits = join_max<ES>(bits, raw[i]);
    }
    if (ES == 2) bits = max(bits & 0xffffu, bits >> 16);
    bits = __reduce_max_sync(0xffffffffu, bits);
    const bool wild = bits >= (ES == 4 ? 0x7f800000u : p.dt == WG_DT_F16 ? 0x7c00u : 0x7f80u);
    float amax = ES == 4 ? __uint_as_float(bits) : dt_unpack2(p.dt, bits).x;
    if (wild) {  // something is not finite: the largest of the rest
      amax = 0.f;
      for (int b0 = held;;) {
#pragma unroll 1
        for (int i = 0; i < APPEND_HOLD; i++) {
          const int tok = b0 + i * tok_step;
          float x[EPL];
          values16<ES>(tok + sub < len ? load16<ES>(src, from + tok * ld, vec) : make_uint4(0, 0, 0, 0), p.dt, x);
#pragma unroll
          for (int k = 0; k < EPL; k++) {
            const float a = fabsf(x[k]);
            if (a <= 3.402823466e38f) amax = fmaxf(amax, a);
          }
        }
        if (b0 == 0) break;
        b0 -= block_len;
      }
      amax = warp_max(amax);
    }
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
    for (int b0 = held;;) {  // the block that is held, then the earlier ones
#pragma unroll
      for (int i = 0; i < APPEND_HOLD; i++) {
        const int tok = b0 + i * tok_step + sub;
        if (tok < len) {
          float x[EPL];
          values16<ES>(raw[i], p.dt, x);
          if (wild) {
#pragma unroll
            for (int k = 0; k < EPL; k++) x[k] = tame(x[k], scale);
          }
          uint32_t out[EPL / 4];
#pragma unroll
          for (int k = 0; k < EPL / 4; k++) out[k] = codes4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3], inv);
          int8_t* to = codes + (int64_t)(first + tok) * p.D + d;
          if constexpr (EPL == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
          else *reinterpret_cast<uint32_t*>(to) = out[0];
        }
      }
      if (b0 == 0) break;
      b0 -= block_len;
      load(b0);
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
  int n, per_cta, units;  // tokens, tokens a CTA takes, (K|V, head) pairs
};
constexpr int READ_WARPS = 8;

// One warp per (K or V, head) and a CTA's tokens, 16 output bytes a lane: the
// codes of consecutive slots are contiguous, and so are a head's values in a row.
template <int ES>
__global__ void __launch_bounds__(READ_WARPS * 32) read_kernel(ReadArgs p) {
  pdl_trigger();
  pdl_wait();
  constexpr int EPL = 16 / ES;
  const int per_tok = p.D / EPL, tok_step = 32 / per_tok, page = 1 << p.shift;
  const int lane = threadIdx.x & 31, unit = blockIdx.y * READ_WARPS + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const int sub = lane / per_tok, d = (lane % per_tok) * EPL;
  const int kv = unit >= p.H, head = unit - kv * p.H;
  void* dst = kv ? p.v : p.k;
  const int64_t ld = kv ? p.ldv : p.ldk, col = (int64_t)head * p.D + d;
  const bool vec = kv ? p.vecv : p.veck;
  const int t0 = blockIdx.x * p.per_cta, t1 = min(p.n, t0 + p.per_cta);
  constexpr int U = 4;  // tokens in flight: their slots, then their codes and scales, then the stores
  for (int tb = t0 + sub; tb < t1; tb += U * tok_step) {
    int slot[U];
#pragma unroll
    for (int i = 0; i < U; i++) slot[i] = tb + i * tok_step < t1 ? __ldg(p.slots + tb + i * tok_step) : -1;
    uint32_t c[U][EPL / 4];
    float scale[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (slot[i] >= p.num_slots) slot[i] = -1;
      const int at = max(slot[i], 0);  // no token: a page that exists is read and nothing is written
      const int64_t block = ((int64_t)(at >> p.shift) * 2 + kv) * p.H + head;
      scale[i] = __ldg(p.scales + block);
      const int8_t* src = p.codes + (block * page + (at & (page - 1))) * p.D + d;
      if constexpr (EPL == 8) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
        c[i][0] = v.x;
        c[i][1] = v.y;
      } else {
        c[i][0] = __ldg(reinterpret_cast<const uint32_t*>(src));
      }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (slot[i] < 0) continue;  // the row stays as it was
      // code + 128 in the low byte of 2^23: exact
      float x[EPL];
#pragma unroll
      for (int k = 0; k < EPL; k++)
        x[k] = (__uint_as_float(__byte_perm(c[i][k >> 2] ^ 0x80808080u, 0x4b000000u, 0x7540 + (k & 3))) - 8388736.f) *
               scale[i];
      const int64_t at = (int64_t)(tb + i * tok_step) * ld + col;
      if (!vec) {
#pragma unroll
        for (int k = 0; k < EPL; k++) dt_store(dst, at + k, p.dt, x[k]);
      } else if constexpr (ES == 4) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + at) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dst) + at) =
            make_uint4(dt_pack2(p.dt, x[0], x[1]), dt_pack2(p.dt, x[2], x[3]), dt_pack2(p.dt, x[4], x[5]),
                       dt_pack2(p.dt, x[6], x[7]));
      }
    }
  }
}

constexpr int KV8_MAX_ROWS = 1 << 30;  // tokens of one call

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

int launch_kv8_append(const wg_kv8& c, const Kv8Rows& r, const int32_t* slots, int n, cudaStream_t st) {
  const int dt = r.dtype;
  AppendArgs a{c.codes, c.scales, c.num_pages * c.page, log2_of(c.page), c.n_kv_head, c.head_dim, r.k, r.v, r.ldk, r.ldv,
               r.head_step, r.batch_step, r.batch, dt, r.veck, r.vecv, slots, n, 1, 2 * c.n_kv_head, APPEND_WARPS};
  // tokens a CTA looks through: few, so that short calls spread over the SMs
  // (every token may begin a run of its own), up to 64 where that leaves
  // enough CTAs
  const int per8 = (a.units + APPEND_WARPS - 1) / APPEND_WARPS;
  while (a.chunk < APPEND_CHUNK && (int64_t)(n / (2 * a.chunk)) * per8 >= 148 * 4) a.chunk *= 2;
  // two pairs a warp where that still leaves waves of CTAs: the search for the
  // runs is shared (96000 tokens 162 -> 150 us; 3800 tokens 11.4 -> 12.3 us,
  // so not there)
  const int per16 = (a.units + 2 * APPEND_WARPS - 1) / (2 * APPEND_WARPS);
  if (a.chunk == APPEND_CHUNK && (int64_t)(n / a.chunk) * per16 >= 148 * 8) a.group = 2 * APPEND_WARPS;
  const int gy = (a.units + a.group - 1) / a.group;
  const dim3 grid((n + a.chunk - 1) / a.chunk, gy), block(APPEND_WARPS * 32);
  return launch_check(dt == WG_DT_F32 ? launch_k(append_kernel<4>, grid, block, 0, st, a)
                                      : launch_k(append_kernel<2>, grid, block, 0, st, a),
                      "kv8_append");
}

}  // namespace wg

extern "C" int wg_kv8_append(const wg_kv8* cache, const void* k, const void* v, int dtype, int64_t ldk, int64_t ldv,
                             const int32_t* slots, int n, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_kv8_append";
  WG_CHECK(kv8_check(what, cache));
  if (!dt_ok(dtype) || n < 0 || n > KV8_MAX_ROWS || (n > 0 && !slots) || !aligned4(slots)) {
    set_error("%s: bad argument (dtype %d, n %d, slots null or misaligned)", what, dtype, n);
    return WG_ERR_INVALID;
  }
  if (n == 0) return WG_OK;
  bool vk, vv;
  const int64_t width = (int64_t)cache->n_kv_head * cache->head_dim;
  WG_CHECK(rows_check(what, "k", k, dtype, ldk, width, &vk));
  WG_CHECK(rows_check(what, "v", v, dtype, ldv, width, &vv));
  OpDevice dev;
  WG_CHECK(dev.enter(what, device));
  const Kv8Rows rows{k, v, ldk, ldv, cache->head_dim, 0, n, dtype, vk, vv};
  return launch_kv8_append(*cache, rows, slots, n, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int wg_kv8_read(const wg_kv8* cache, const int32_t* slots, int n, void* k, void* v, int dtype, int64_t ldk,
                           int64_t ldv, int device, void* stream) {
  using namespace wg;
  const char* what = "wg_kv8_read";
  WG_CHECK(kv8_check(what, cache));
  if (!dt_ok(dtype) || n < 0 || n > KV8_MAX_ROWS || (n > 0 && !slots) || !aligned4(slots)) {
    set_error("%s: bad argument (dtype %d, n %d, slots null or misaligned)", what, dtype, n);
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
             cache->head_dim, k, v, ldk, ldv, dtype, vk, vv, slots, n, 4,
               2 * cache->n_kv_head};
  // tokens a CTA: few where calls are short, up to 32 where there are CTAs enough
  const int gy = (a.units + READ_WARPS - 1) / READ_WARPS;
  while (a.per_cta < 32 && (int64_t)(n / (2 * a.per_cta)) * gy >= 148 * 8) a.per_cta *= 2;
  const dim3 grid((n + a.per_cta - 1) / a.per_cta, gy);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return launch_check(dtype == WG_DT_F32 ? launch_k(read_kernel<4>, grid, dim3(256), 0, st, a)
                                         : launch_k(read_kernel<2>, grid, dim3(256), 0, st, a),
                      "kv8_read");
}
