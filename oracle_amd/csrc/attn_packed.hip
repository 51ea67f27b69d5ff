// Causal attention over whole prompts packed one behind the other (orc_attention_packed), grouped heads, bf16 / fp16.
//
// out[t] = sum_j p_j v_j / sum_j p_j, p_j = exp2(c (q_t . k_j - m)), c = scale * log2(e), j over the tokens 0..t of t's sequence, with the running
// maximum m and sum of one pass over the keys (flash32.h). One workgroup = NW waves x 32 query rows of one head; K / V tiles of 64 keys
// arrive by LDS-DMA in a 2-deep ring: wait for the tile -> barrier -> issue the next one's DMA -> compute.
#include <algorithm>
#include <type_traits>

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

template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void packed_kernel(PackedArgs a) {
  typedef Tile64<HD> Tile;
  constexpr int KB = 64, NT = 256;
  constexpr int RND = KB * Tile::CH / NT;    // DMA instructions per wave, operand and tile
  constexpr int KPR = NT / Tile::CH;         // keys one round of them covers
  __shared__ __attribute__((aligned(16))) char smem[4 * Tile::BYTES];   // K of even and odd tiles, V of even and odd tiles
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
  const T* kb = (const T*)a.k + (size_t)seq * a.k_ts + (size_t)kvh * a.k_hs;
  const T* vb = (const T*)a.v + (size_t)seq * a.v_ts + (size_t)kvh * a.v_hs;
  const int qw = q0 + w * 32, qrow = qw + (lane & 31);
  Flash32<T, HD> f;
  f.init((const T*)a.q + (size_t)(seq + (qrow < len ? qrow : len - 1)) * a.q_ts + (size_t)head * a.q_hs, lane);
  const int k_end = q0 + ROWS < len ? q0 + ROWS : len;

  // Lane p of round r fills chunk p % CH of key r KPR + p / CH. The swizzle looks at the key's low bits only, which the rounds share.
  const int key_p = tid / Tile::CH, ch_p = tid % Tile::CH;
  const int ck = Tile::swz_k(key_p, ch_p) * 8, cv = Tile::swz_v(key_p, ch_p) * 8;
  static_assert(KPR % 16 == 0, "the swizzle repeats every 16 keys");
  const unsigned koff = (unsigned)(key_p * a.k_ts + ck), voff = (unsigned)(key_p * a.v_ts + cv);
  auto dma = [&](const T* base, long ts, unsigned off, int c, int k0, char* to) {
    to += w * 1024;
    if (k0 + KB <= len) {
      const T* from = base + (size_t)k0 * ts;
#pragma unroll
      for (int r = 0; r < RND; ++r)
        __builtin_amdgcn_global_load_lds((glb_void_t*)(from + (size_t)r * KPR * ts + off), (lds_void_t*)(to + r * NT * 16), 16, 0, 0);
    } else {
#pragma unroll
      for (int r = 0; r < RND; ++r) {
        int src = k0 + r * KPR + key_p;
        src = src < len ? src : len - 1;   // behind the last token: that token again, its score is masked
        __builtin_amdgcn_global_load_lds((glb_void_t*)(base + (size_t)src * ts + c), (lds_void_t*)(to + r * NT * 16), 16, 0, 0);
      }
    }
  };
  auto dma_k = [&](int k0, int stage) { dma(kb, a.k_ts, koff, ck, k0, smem + stage * Tile::BYTES); };
  auto dma_v = [&](int k0, int stage) { dma(vb, a.v_ts, voff, cv, k0, smem + (2 + stage) * Tile::BYTES); };
  // One iteration a tile t: wait for its values and the next tile's keys, barrier (the waves are through with the tile before), ask for what comes
  // behind those. PAR = t % 2.
  const int tiles = (k_end + KB - 1) / KB;
  auto advance = [&](int t, auto par) {
    constexpr int PAR = decltype(par)::value;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 2 < tiles) dma_k((t + 2) * KB, PAR);
    if (t + 1 < tiles) dma_v((t + 1) * KB, PAR ^ 1);
  };
  float tm = 0.f;
  // tile t, whose scores are in s: the next tile's scores (to n) between this one's exponentials, then this one's values
  auto step = [&](int t, const f32x16 (&s)[2], f32x16 (&n)[2], auto par) {
    constexpr int PAR = decltype(par)::value;
    advance(t, par);
    f.raise(tm, a.c);
    const float mc = f.base(a.c);
    const char* sK = smem + (PAR ^ 1) * Tile::BYTES;
    u32x4 pf[4];
    n[0] = f.scores(sK, 0);
    f.weights(s[0], a.c, mc, pf);
    n[1] = f.scores(sK, 1);
    f.weights(s[1], a.c, mc, pf + 2);
    f.values(smem + (2 + PAR) * Tile::BYTES, pf);
    tm = f.largest(n);
  };
  // the wave's last tile, the only one with keys in a query's future: tiles are 64 keys, the wave's queries 32 from a multiple of 32 on
  auto finish = [&](int t, f32x16 (&s)[2], auto par) {
    constexpr int PAR = decltype(par)::value;
    advance(t, par);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (t * KB + Flash32<T, HD>::key_of(b, i, h) > qrow) s[b][i] = -INFINITY;
    f.add(smem + (2 + PAR) * Tile::BYTES, s, a.c);
  };
  typedef std::integral_constant<int, 0> even;
  typedef std::integral_constant<int, 1> odd;
  dma_k(0, 0);
  dma_v(0, 0);
  if (tiles > 1) {
    dma_k(KB, 1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * RND) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RND) : "memory");
  }
  __syncthreads();
  const int mine = qw >= len ? 0 : (qw + 31) / KB + 1;   // the wave's tiles: those behind are all in its future; 0: it has no query
  int t = 0;
  if (mine) {
    f32x16 s[2] = {f.scores(smem, 0), f.scores(smem, 1)}, n[2];
    tm = f.largest(s);
    for (; t + 2 < mine; t += 2) {
      step(t, s, n, even());
      step(t + 1, n, s, odd());
    }
    if (t + 1 < mine) {
      step(t, s, n, even());
      finish(t + 1, n, odd());
    } else {
      finish(t, s, even());
    }
  }
  for (t = mine; t < tiles; ++t) {   // the other waves' tiles
    if (t & 1) advance(t, odd());
    else advance(t, even());
  }
  const float inv = 1.0f / f.total();
  if (qrow >= len) return;
  T* op = (T*)a.o + (size_t)(seq + qrow) * a.o_ts + (size_t)head * a.o_hs;
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      u32x2 st = {cvt2<T>(f.o[dt][i] * inv, f.o[dt][i + 1] * inv), cvt2<T>(f.o[dt][i + 2] * inv, f.o[dt][i + 3] * inv)};
      *(u32x2*)(op + dt * 32 + 2 * i + 4 * h) = st;
    }
}

template <typename T, int HD> void launch_hd(const PackedArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_kernel<T, HD>), dim3((unsigned)(a.n_work * a.hq)), dim3(256), 0, s, a);
}

}  // namespace

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
  // a prompt's tiles together, so that its K / V are read from L2 by all of them; long prompts first, and in a prompt the tiles with the most keys
  std::sort(w, w + at, [](const int4& x, const int4& y) { return x.y != y.y ? x.y > y.y : x.x != y.x ? x.x < y.x : x.z > y.z; });
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
  if ((int64_t)n_work * n_heads > 0x7fffffff) return orc_fail(who, "too many tiles");
  for (int i = 0; i < 8; ++i)
    if (st[i] < 0 || st[i] % 8) return orc_fail(who, "strides are not multiples of 8 elements");
  if (st[2] >= 1 << 24 || st[4] >= 1 << 24) return orc_fail(who, "K / V token strides of 2^24 elements and more");   // a tile's offsets are 32-bit
  if (n_work == 0) return 0;
  if (!q || !k || !v || !out || !work) return orc_fail(who, "null argument");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)work) & 15) return orc_fail(who, "tensors are not aligned to 16 bytes");
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
