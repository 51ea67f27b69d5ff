// Causal attention over whole prompts packed one behind the other (orc_attention_packed), grouped heads, bf16 / fp16.
//
// out[t] = sum_j p_j v_j / sum_j p_j, p_j = exp2(c (q_t . k_j - m)), c = scale * log2(e), j over the tokens 0..t of t's sequence, with the running
// maximum m and sum of one pass over the keys (flash32.h). One workgroup = 4 waves x 32 query rows of one head.
//
// Long prompts are bound by the matrix cores and the softmax beside them, at the clock that the power limit leaves (about 1.75 GHz): 2 prompts of 15k
// and 24k tokens, 32 heads on 8, head dim 128, 5.8 ms = 1130 TFLOP/s (5.55 to 5.95 ms on different cards), 0.88 of an 8192^3 bf16 product. Short ones by
// what a tile costs before its first product (Q, then two K images from HBM) and by the uneven end: 8 prompts of 640..900, 32 heads, 68 us (570 TFLOP/s,
// 3.0 TB/s); 48 of 0..2304, 16 heads on 4, head dim 64, fp16, 164 us (690 TFLOP/s: half the products to a tile's exponentials). Medians of 200 launches one
// behind the other (40 of the long ones): the first ms of them is faster (157 us a launch of the last case), the next 20 ms up to a third slower, until
// the clock has settled under the power limit.
// 128 rows a workgroup and not 256: those halve the reads of K / V, which L2 serves anyway, and leave fewer tiles to spread (measured slower).
// Two workgroups fit a CU at head dim 128 (256 registers a lane), three at 64 (168).
#include <algorithm>
#include <cstdlib>

#include "../../include/oracle_hip.h"
#include "kernels.h"
#include "flash32.h"

namespace {

constexpr int ROWS = 128;   // query rows of a tile: 4 waves of 32

struct PackedArgs {
  const char *q, *k, *v;
  char* o;
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;   // elements
  const int4* work;
  int n_work, total, hq, group;
  float c;   // scale * log2(e)
};

// where the tiles come from and what a wave may see of them (flash_loop)
template <typename T, int HD> struct PackedSrc {
  typedef Tile64<HD> Tile;
  static constexpr int RND = Tile::KEYS * Tile::CH / 256;    // DMA instructions per wave and image
  static constexpr int KPR = 256 / Tile::CH;                 // keys one round of them covers
  static_assert(KPR % 16 == 0, "the swizzle repeats every 16 keys: the rounds share it");
  const T *kb, *vb;
  long k_ts, v_ts;
  int len, qrow, w, h;
  int koff, voff;                        // bytes, of the lane in round 0
  __amdgpu_buffer_rsrc_t kr, vr;         // of the tile that is asked for next
  // Lane p of round r fills chunk p % CH of key r KPR + p / CH.
  __device__ __forceinline__ void init(int tid) {
    const int key_p = tid / Tile::CH;
    w = __builtin_amdgcn_readfirstlane(tid >> 6);
    h = (tid & 63) >> 5;
    koff = (int)(key_p * k_ts + Tile::swz_k(key_p, tid % Tile::CH) * 8) * 2;
    voff = (int)(key_p * v_ts + Tile::swz_v(key_p, tid % Tile::CH) * 8) * 2;
  }
  // Buffer descriptors that start at the tile and end with the sequence: what lies behind the last token arrives as zeros, without a test. (The whole
  // offset is in the lane's: a scalar one beyond the end would wrap the range check.)
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(const T* base, long ts, int t) const {
    int left = len - t * Tile::KEYS;
    left = left < Tile::KEYS ? left : Tile::KEYS;
    const int bytes = (int)((left - 1) * ts + HD) * 2;
    return buffer_of(base + (long)t * Tile::KEYS * ts, left > 0 ? bytes : 0);
  }
  __device__ __forceinline__ void next(int t) {
    kr = tile(kb, k_ts, t + 2);
    vr = tile(vb, v_ts, t + 1);
  }
  __device__ __forceinline__ void K(int, int r, char* to) const {
    buffer_load16_lds(kr, koff + (int)(r * KPR * k_ts * 2), to + w * 1024 + r * 4096);
  }
  __device__ __forceinline__ void V(int, int r, char* to) const {
    buffer_load16_lds(vr, voff + (int)(r * KPR * v_ts * 2), to + w * 1024 + r * 4096);
  }
  // Only a wave's last tile has keys in a query's future: tiles are 64 keys, the wave's queries 32 from a multiple of 32 on.
  __device__ __forceinline__ void mask_last(int t, f32x16 (&s)[2]) const {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (t * Tile::KEYS + Flash32<T, HD>::key_of(b, i, h) > qrow) s[b][i] = -INFINITY;
  }
};

template <typename T, int HD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void packed_kernel(PackedArgs a) {
  typedef Tile64<HD> Tile;
  __shared__ __attribute__((aligned(16))) char k0[Tile::BYTES], k1[Tile::BYTES], v0[Tile::BYTES], v1[Tile::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  // Workgroup ids go round robin over the 8 XCDs: where the heads divide by 8 an XCD keeps hq / 8 of them, so the tiles that read the
  // same K / V run on one L2. The plan lists long tiles first.
  int wi, head;
  {
    const int lin = blockIdx.x;
    if ((a.hq & 7) == 0) {
      const int per = a.hq >> 3, slot = lin >> 3;
      head = (lin & 7) * per + slot % per;
      wi = slot / per;
    } else {
      head = lin % a.hq;
      wi = lin / a.hq;
    }
  }
  const int4 wk = a.work[wi];
  const int seq = wk.x, len = wk.y, q0 = wk.z;
  if (seq < 0 || q0 < 0 || len <= q0 || len > a.total - seq) return;   // a plan of other prompts than these
  const int kvh = head / a.group;
  PackedSrc<T, HD> src;
  src.kb = (const T*)a.k + (size_t)seq * a.k_ts + (size_t)kvh * a.k_hs;
  src.vb = (const T*)a.v + (size_t)seq * a.v_ts + (size_t)kvh * a.v_hs;
  src.k_ts = a.k_ts; src.v_ts = a.v_ts; src.len = len;
  const int qw = q0 + w * 32, qrow = qw + (lane & 31);
  src.qrow = qrow;
  src.init(tid);
  Flash32<T, HD> f;
  f.init((const T*)a.q + (size_t)(seq + (qrow < len ? qrow : len - 1)) * a.q_ts + (size_t)head * a.q_hs, lane);
  const int k_end = q0 + ROWS < len ? q0 + ROWS : len;
  const Images im{k0, k1, v0, v1};
  const int tiles = (k_end + Tile::KEYS - 1) / Tile::KEYS;
  const int mine = qw >= len ? 0 : (qw + 31) / Tile::KEYS + 1;   // the wave's tiles: those behind are all in its future; 0: it has no query
  flash_loop(f, src, im, tiles, mine, a.c);
  // A value that is infinite or NaN comes out where it was seen, and in the wave's last tile also where it was masked, as 0 times it. Told by the
  // outputs, and done again one tile at a time with those values apart.
  if (__syncthreads_or(!f.finite())) {
    f.clear();
    for (int t = 0; t < tiles; ++t) {
      __syncthreads();
      src.next(t - 2);
#pragma unroll
      for (int r = 0; r < src.RND; ++r) src.K(t, r, im.k0);
      src.next(t - 1);
#pragma unroll
      for (int r = 0; r < src.RND; ++r) src.V(t, r, im.v0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t >= mine) continue;
      f32x16 s[2] = {f.scores(im.k0, 0), f.scores(im.k0, 1)};
      src.mask_last(t, s);
      f.raise(f.largest(s), a.c);
      const float mc = f.base(a.c);
      u32x4 pf[4];
      f.weights(s[0], a.c, mc, pf);
      f.weights(s[1], a.c, mc, pf + 2);
      f.values_careful(im.v0, pf, qrow - t * Tile::KEYS, lane >> 5);
    }
    __syncthreads();
  }
  T* op = (T*)a.o + (size_t)(seq + qw) * a.o_ts + (size_t)head * a.o_hs;
  const float total = f.total();   // 0: all scores are -inf, the softmax is 0 / 0 (and not 1 / 0, which would pass on an infinity of V)
  f.template rows<false>(im.of(w), lane, total != 0.f ? 1.f / total : NAN, [&](int row, int byte, u32x4 v) {
    if (qw + row < len) *(u32x4*)((char*)(op + (size_t)row * a.o_ts) + byte) = v;
  });
}

template <typename T, int HD> void launch_hd(const PackedArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_kernel<T, HD>), dim3((unsigned)(a.n_work * a.hq)), dim3(256), 0, s, a);
}

// The tiles of up to kMaxRows prompts, by prompt, written on the device; the prompts longest first, first: tiles before each of them. (Without
// the order by keys that orc_attn_plan gives the last quarter: 3 us of a 7B layer's 1900 at 8 prompts of 640..900.)
struct PlanArgs { int n, first[kMaxRows + 1], start[kMaxRows], len[kMaxRows]; };
__global__ __launch_bounds__(256) void plan_kernel(PlanArgs a, int4* work) {
  for (int x = threadIdx.x; x < a.first[a.n]; x += 256) {
    int i = 0;
    while (i + 1 < a.n && x >= a.first[i + 1]) ++i;
    work[x] = int4{a.start[i], a.len[i], (a.first[i + 1] - 1 - x) * ROWS, 0};
  }
}

}  // namespace

bool views_meet(HeadView a, HeadView b) {
  for (HeadView* x : {&a, &b}) {
    if (x->tokens < 1) return false;
    if (x->tokens == 1) x->ts = 0;   // the stride of one element does not matter
    if (x->heads == 1) x->hs = 0;
  }
  const int64_t d0 = ((intptr_t)b.p - (intptr_t)a.p) / 2;   // both start on 16 bytes
  const int64_t end_a = (a.tokens - 1) * a.ts + (a.heads - 1) * a.hs + a.hd, end_b = (b.tokens - 1) * b.ts + (b.heads - 1) * b.hs + b.hd;
  if (d0 >= end_a || -d0 >= end_b) return false;
  if (a.tokens > 1 && b.tokens > 1 && a.ts != b.ts) return true;
  const int64_t ts = a.tokens > 1 ? a.ts : b.ts, row_a = (a.heads - 1) * a.hs + a.hd, row_b = (b.heads - 1) * b.hs + b.hd;
  if (ts > 0) {   // slices of one projection's rows: b's part of a row behind a's
    const int64_t at = (d0 % ts + ts) % ts;
    if (at >= row_a && at + row_b <= ts) return false;
  }
  // heads d apart, tokens k apart: closest for the two k around -d / ts
  auto close = [&](int64_t d) {
    const int64_t lo = -(a.tokens - 1), hi = b.tokens - 1, k0 = ts > 0 ? -d / ts : 0;
    for (int64_t k = k0 - 1; k <= k0 + 1; ++k)
      if (std::abs(d + std::min(std::max(k, lo), hi) * ts) < std::max(a.hd, b.hd)) return true;
    return false;
  };
  const bool same = a.hs == b.hs || a.heads == 1 || b.heads == 1;
  const int64_t hs = a.heads > 1 ? a.hs : b.hs;
  if (same) {
    for (int64_t h = -(int64_t)(a.heads - 1); h < b.heads; ++h)
      if (close(d0 + h * hs)) return true;
    return false;
  }
  for (int64_t x = 0; x < a.heads; ++x)
    for (int64_t y = 0; y < b.heads; ++y)
      if (close(d0 + y * b.hs - x * a.hs)) return true;
  return false;
}

bool out_meets_q(const HeadView& o, const HeadView& q) {
  if (o.p == q.p && (o.tokens <= 1 || o.ts == q.ts) && (o.heads == 1 || o.hs == q.hs)) return false;
  return views_meet(o, q);
}

int attn_plan_ints(int rows) { return (rows / ROWS + kMaxRows) * 4; }

int launch_attn_plan(const PackedRows& p, int32_t* work, hipStream_t s) {
  if (p.n < 1 || p.n > kMaxRows) return orc_fail("launch_attn_plan", "1..32 prompts");
  PlanArgs a;
  int order[kMaxRows];
  for (int i = 0; i < p.n; ++i) order[i] = i;
  std::sort(order, order + p.n, [&](int x, int y) {
    const int lx = p.start[x + 1] - p.start[x], ly = p.start[y + 1] - p.start[y];
    return lx != ly ? lx > ly : x < y;
  });
  a.n = p.n;
  a.first[0] = 0;
  for (int i = 0; i < p.n; ++i) {
    a.start[i] = p.start[order[i]];
    a.len[i] = p.start[order[i] + 1] - a.start[i];
    a.first[i + 1] = a.first[i] + (a.len[i] + ROWS - 1) / ROWS;
  }
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(256), 0, s, a, (int4*)work);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? a.first[a.n] : orc_fail("launch_attn_plan", hipGetErrorString(e));
}

extern "C" int orc_attn_plan(const int32_t* lens, int n, int32_t* out, int capacity) {
  if (n < 0 || (n > 0 && !lens)) return orc_fail("orc_attn_plan", "null argument");
  int64_t tiles = 0, start = 0;
  for (int i = 0; i < n; ++i) {
    if (lens[i] < 0) return orc_fail("orc_attn_plan", "negative length");
    start += lens[i];
    tiles += ((int64_t)lens[i] + ROWS - 1) / ROWS;
  }
  if (start > 0x7fffffff) return orc_fail("orc_attn_plan", "more than 2^31 - 1 tokens");
  if (!out) return (int)tiles;
  if (tiles > capacity) return orc_fail("orc_attn_plan", "capacity too small");
  int4* w = (int4*)out;
  int at = 0, first = 0;
  for (int i = 0; i < n; first += lens[i], ++i)
    for (int q0 = 0; q0 < lens[i]; q0 += ROWS) w[at++] = int4{first, lens[i], q0, 0};
  // A prompt's tiles together, so that its K / V are read from L2 by all of them; long prompts first, and in a prompt the tiles with the most keys.
  // The last quarter of all tiles by their keys alone, so that no long one starts near the end (8 prompts of 640..900 tokens: all by prompt
  // 65 us, the last quarter by keys 62, all by keys 76).
  std::sort(w, w + at, [](const int4& x, const int4& y) { return x.y != y.y ? x.y > y.y : x.x != y.x ? x.x < y.x : x.z > y.z; });
  std::sort(w + at - at / 4, w + at, [](const int4& x, const int4& y) {
    const int kx = std::min(x.z + ROWS, x.y), ky = std::min(y.z + ROWS, y.y);
    return kx != ky ? kx > ky : x.x < y.x;
  });
  return at;
}

extern "C" int orc_attention_packed(const void* q, const void* k, const void* v, void* out, const int64_t* st, const int32_t* work, int n_work,
                                    int total, int n_heads, int n_kv_heads, int head_dim, int dtype, float scale, void* stream) {
  const char* who = "orc_attention_packed";
  if (!st || n_work < 0 || total < 0) return orc_fail(who, "bad argument");
  if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads) return orc_fail(who, "n_heads is not a multiple of n_kv_heads");
  if (head_dim != 64 && head_dim != 128) return orc_fail(who, "head_dim is 64 or 128");
  if (dtype != 0 && dtype != 1) return orc_fail(who, "dtype is 0 (bf16) or 1 (fp16)");
  if (!(scale > 0.f) || !(scale < 1e30f)) return orc_fail(who, "scale is not positive and finite");
  if ((int64_t)n_work * n_heads > 0xffffff) return orc_fail(who, "too many tiles: with the heads 2^24 - 1 at the most");   // 256 threads each: 32 bits
  for (int i = 0; i < 8; ++i)
    if (st[i] < 0 || st[i] % 8) return orc_fail(who, "strides are not multiples of 8 elements");
  if (st[2] >= 1 << 24 || st[4] >= 1 << 24) return orc_fail(who, "K / V token strides of 2^24 elements and more");   // a tile's offsets are 32-bit
  if (n_work == 0) return 0;
  if (!q || !k || !v || !out || !work) return orc_fail(who, "null argument");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)work) & 15) return orc_fail(who, "tensors are not aligned to 16 bytes");
  const HeadView vo{out, st[6], st[7], total, n_heads, head_dim};
  if (views_meet(vo, {k, st[2], st[3], total, n_kv_heads, head_dim}) || views_meet(vo, {v, st[4], st[5], total, n_kv_heads, head_dim}))
    return orc_fail(who, "out lies over k or v");
  if (out_meets_q(vo, {q, st[0], st[1], total, n_heads, head_dim})) return orc_fail(who, "out lies over q and is not q");
  PackedArgs a;
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.o = (char*)out;
  a.q_ts = st[0]; a.q_hs = st[1]; a.k_ts = st[2]; a.k_hs = st[3]; a.v_ts = st[4]; a.v_hs = st[5]; a.o_ts = st[6]; a.o_hs = st[7];
  a.work = (const int4*)work; a.n_work = n_work; a.total = total; a.hq = n_heads; a.group = n_heads / n_kv_heads;
  a.c = scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) head_dim == 128 ? launch_hd<__bf16, 128>(a, s) : launch_hd<__bf16, 64>(a, s);
  else head_dim == 128 ? launch_hd<_Float16, 128>(a, s) : launch_hd<_Float16, 64>(a, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : orc_fail(who, hipGetErrorString(e));
}
