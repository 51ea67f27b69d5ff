// Causal attention over whole prompts packed one behind the other (orc_attention_packed), grouped heads, bf16 / fp16.
//
// out[t] = sum_j p_j v_j / sum_j p_j, p_j = exp2(c (q_t . k_j - m)), c = scale * log2(e), j over the tokens 0..t of t's sequence, with the running
// maximum m and sum of one pass over the keys (flash32.h). One workgroup = NW waves x 32 query rows of one head; K / V tiles of 64 keys
// arrive by LDS-DMA in a 2-deep ring: wait for the tile -> barrier -> issue the next one's DMA -> compute.
#include <stdlib.h>
#include <algorithm>
#include <type_traits>

#include "../../include/oracle_hip.h"
#include "kernels.h"
#include "flash32.h"

namespace {

struct PackedArgs {
  const char *q, *k, *v;
  char* o;
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;   // elements
  const int4* work;
  int n_work, total, hq, group;
  float c;   // scale * log2(e)
};

template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64, 2) void packed_kernel(PackedArgs a) {
  typedef Tile64<HD> Tile;
  constexpr int KB = 64, NT = NW * 64;
  constexpr int RND = KB * Tile::CH / NT;    // DMA instructions per wave, operand and tile
  constexpr int KPR = NT / Tile::CH;         // keys one round of them covers
  __shared__ __attribute__((aligned(16))) char smem[4 * Tile::BYTES];   // [stage][K | V]
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
  const int k_end = q0 + NW * 32 < len ? q0 + NW * 32 : len;

  // Lane p of round r fills chunk p % CH of key r KPR + p / CH. The swizzle looks at the key's low bits only, which the rounds share.
  const int key_p = tid / Tile::CH, ch_p = tid % Tile::CH;
  const int ck = Tile::swz_k(key_p, ch_p) * 8, cv = Tile::swz_v(key_p, ch_p) * 8;
  static_assert(KPR % 16 == 0, "the swizzle repeats every 16 keys");
  const unsigned koff = (unsigned)(key_p * a.k_ts + ck), voff = (unsigned)(key_p * a.v_ts + cv);
  auto dma = [&](int k0, int stage) {
    char* sk = smem + stage * 2 * Tile::BYTES + w * 1024;
    if (k0 + KB <= len) {
      const T* kr = kb + (size_t)k0 * a.k_ts;
      const T* vr = vb + (size_t)k0 * a.v_ts;
#pragma unroll
      for (int r = 0; r < RND; ++r) {
        __builtin_amdgcn_global_load_lds((glb_void_t*)(kr + (size_t)r * KPR * a.k_ts + koff), (lds_void_t*)(sk + r * NT * 16), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_void_t*)(vr + (size_t)r * KPR * a.v_ts + voff), (lds_void_t*)(sk + Tile::BYTES + r * NT * 16), 16, 0, 0);
      }
    } else {
#pragma unroll
      for (int r = 0; r < RND; ++r) {
        int src = k0 + r * KPR + key_p;
        src = src < len ? src : len - 1;   // behind the last token: that token again, its score is masked
        __builtin_amdgcn_global_load_lds((glb_void_t*)(kb + (size_t)src * a.k_ts + ck), (lds_void_t*)(sk + r * NT * 16), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_void_t*)(vb + (size_t)src * a.v_ts + cv), (lds_void_t*)(sk + Tile::BYTES + r * NT * 16), 16, 0, 0);
      }
    }
  };
  auto step = [&](int k0, auto st) {
    constexpr int stage = decltype(st)::value;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + KB < k_end) dma(k0 + KB, stage ^ 1);
    if (k0 > qw + 31) return;   // all of the tile is in this wave's future
    const char* sK = smem + stage * 2 * Tile::BYTES;
    f32x16 s[2];
    f.scores(sK, s);
    if (k0 + KB - 1 > qw) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + Flash32<T, HD>::key_of(b, i, h) > qrow) s[b][i] = -INFINITY;
    }
    f.add(sK + Tile::BYTES, s, a.c);
  };
  dma(0, 0);
  for (int k0 = 0; k0 < k_end; k0 += 2 * KB) {
    step(k0, std::integral_constant<int, 0>());
    if (k0 + KB < k_end) step(k0 + KB, std::integral_constant<int, 1>());
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

template <typename T, int HD> void launch_nw(const PackedArgs& a, int bm, hipStream_t s) {
  const dim3 grid((unsigned)(a.n_work * a.hq));
  if (bm == 256) hipLaunchKernelGGL((packed_kernel<T, HD, 8>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((packed_kernel<T, HD, 4>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" int orc_attn_plan(const int32_t* lens, int n, int bm, int32_t* out, int capacity) {
  if (n < 0 || (n > 0 && !lens)) return orc_fail("orc_attn_plan", "null argument");
  if (bm != 128 && bm != 256) return orc_fail("orc_attn_plan", "tile height is 128 or 256");
  int64_t tiles = 0, start = 0;
  for (int i = 0; i < n; ++i) {
    if (lens[i] < 0) return orc_fail("orc_attn_plan", "negative length");
    start += lens[i];
    tiles += ((int64_t)lens[i] + bm - 1) / bm;
  }
  if (start > 0x7fffffff) return orc_fail("orc_attn_plan", "more than 2^31 - 1 tokens");
  if (!out) return (int)tiles;
  if (tiles > capacity) return orc_fail("orc_attn_plan", "capacity too small");
  int4* w = (int4*)out;
  int at = 0, first = 0;
  for (int i = 0; i < n; first += lens[i], ++i)
    for (int q0 = 0; q0 < lens[i]; q0 += bm) w[at++] = int4{first, lens[i], q0, 0};
  const bool lpt = getenv("LPT") != nullptr;
  std::sort(w, w + at, [bm,lpt](const int4& x, const int4& y) {
    if (lpt) {
    const int kx = std::min(x.z + bm, x.y), ky = std::min(y.z + bm, y.y);
    return kx != ky ? kx > ky : x.x != y.x ? x.x < y.x : x.z < y.z;
    }
    return x.y != y.y ? x.y > y.y : x.x != y.x ? x.x < y.x : x.z > y.z;
  });
  return at;
}

extern "C" int orc_attn_tile(const int32_t* lens, int n, int n_heads) {
  if (getenv("BMX")) return atoi(getenv("BMX"));
  return 128;
}

extern "C" int orc_attention_packed(const void* q, const void* k, const void* v, void* out, const int64_t* st, const int32_t* work, int n_work,
                                    int bm, int total, int n_heads, int n_kv_heads, int head_dim, int dtype, float scale, void* stream) {
  const char* who = "orc_attention_packed";
  if (!st || n_work < 0 || total < 0) return orc_fail(who, "bad argument");
  if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads) return orc_fail(who, "n_heads is not a multiple of n_kv_heads");
  if (head_dim != 64 && head_dim != 128) return orc_fail(who, "head_dim is 64 or 128");
  if (dtype != 0 && dtype != 1) return orc_fail(who, "dtype is 0 (bf16) or 1 (fp16)");
  if (bm != 128 && bm != 256) return orc_fail(who, "tile height is 128 or 256");
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
  if (dtype == 0) head_dim == 128 ? launch_nw<__bf16, 128>(a, bm, s) : launch_nw<__bf16, 64>(a, bm, s);
  else head_dim == 128 ? launch_nw<_Float16, 128>(a, bm, s) : launch_nw<_Float16, 64>(a, bm, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : orc_fail(who, hipGetErrorString(e));
}
