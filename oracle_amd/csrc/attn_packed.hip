// Causal attention over whole prompts packed one behind the other (orc_attention_packed), grouped heads, bf16 / fp16.
//
// out[t] = sum_j p_j v_j / sum_j p_j, p_j = exp2(c (q_t . k_j - m)), c = scale * log2(e), j over the tokens 0..t of t's sequence, with the running
// maximum m and sum of one pass over the keys. Orientation (no value crosses lanes between the two products):
//   S^T = K . Q^T    A = 32 keys x 16 from LDS, B = the wave's 32 query columns held in registers
//                    -> lane (q = lane & 31, h = lane >> 5) holds keys 8 (i / 4) + 4 h + i % 4 of its query, i = 0..15
//   O^T = V^T . P^T  the k-slots (h, j) of the product are DEFINED as the keys the lane holds: P is its own registers rounded to 16 bits,
//                    V^T comes by the transposing LDS read in that order.
// One workgroup = NW waves x 32 query rows of one head; K / V tiles of 64 keys by LDS-DMA into a 2-deep ring.
#include <algorithm>

#include "../../include/oracle_hip.h"
#include "kernels.h"
#include "mma16.h"

namespace {

struct PackedArgs {
  const char *q, *k, *v;
  char* o;
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;   // elements
  const int4* work;
  int n_work, total, hq, group;
  float c;   // scale * log2(e)
};

// 16-byte chunk of a K / V row image -> place inside the row (an involution), chosen so that the 16 lanes of a ds_read_b128 phase (16 keys, one
// chunk) and the 4 keys x 64 bytes of half a transposing read fall on different banks
template <int HD> __device__ __forceinline__ int swz_k(int key, int ch) { return HD == 128 ? ch ^ (key & 15) : ch ^ ((key >> 1) & 7); }
template <int HD> __device__ __forceinline__ int swz_v(int key, int ch) { return HD == 128 ? ch ^ ((key & 3) << 2) : ch ^ (((key >> 1) & 1) << 2); }

template <typename T, int HD, int NW>
__global__ __launch_bounds__(NW * 64, NW == 8 ? 2 : 2) void packed_kernel(PackedArgs a) {
  typedef typename Mma<T>::v8 v8;
  constexpr int KB = 64, ROWB = HD * 2, CH = HD / 8, TILE = KB * ROWB, NT = NW * 64;
  constexpr int RND = KB * CH / NT;    // DMA instructions per wave, operand and tile
  constexpr int KPR = NT / CH;         // keys one round of them covers
  __shared__ __attribute__((aligned(16))) char smem[4 * TILE];   // [stage][K | V]
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c32 = lane & 31, h = lane >> 5;
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
  const T* qb = (const T*)a.q + (size_t)seq * a.q_ts + (size_t)head * a.q_hs;
  const T* kb = (const T*)a.k + (size_t)seq * a.k_ts + (size_t)kvh * a.k_hs;
  const T* vb = (const T*)a.v + (size_t)seq * a.v_ts + (size_t)kvh * a.v_hs;
  const int qw = q0 + w * 32, qrow = qw + c32;
  v8 qf[HD / 16];
  {
    const T* qp = qb + (size_t)(qrow < len ? qrow : len - 1) * a.q_ts + h * 8;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) qf[kk] = *(const v8*)(qp + kk * 16);
  }
  const int k_end = q0 + NW * 32 < len ? q0 + NW * 32 : len;

  const int key_p = tid / CH, ch_p = tid % CH;
  auto dma = [&](int k0, int stage) {
    char* sk = smem + stage * 2 * TILE;
#pragma unroll
    for (int r = 0; r < RND; ++r) {
      const int key = r * KPR + key_p;
      const int src = k0 + key < len ? k0 + key : len - 1;   // behind the last token: a token again, its score is masked
      __builtin_amdgcn_global_load_lds((glb_void_t*)(kb + (size_t)src * a.k_ts + swz_k<HD>(key, ch_p) * 8), (lds_void_t*)(sk + (r * NT + w * 64) * 16), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_void_t*)(vb + (size_t)src * a.v_ts + swz_v<HD>(key, ch_p) * 8), (lds_void_t*)(sk + TILE + (r * NT + w * 64) * 16), 16, 0, 0);
    }
  };

  f32x16 o[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  float m = -INFINITY, l = 0.f;   // l: the lane's own keys only, joined with the other half at the end

  dma(0, 0);
  int stage = 0;
  for (int k0 = 0; k0 < k_end; k0 += KB, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + KB < k_end) dma(k0 + KB, stage ^ 1);
    if (k0 > qw + 31) continue;   // all of the tile is in this wave's future
    const char* sK = smem + stage * 2 * TILE;
    const char* sV = sK + TILE;
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] = 0.f;
      const int key = b * 32 + c32;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const v8 kf = *(const v8*)(sK + key * ROWB + (swz_k<HD>(key, kk * 2 + h) << 4));
        s[b] = Mma<T>::m32(kf, qf[kk], s[b]);
      }
    }
    if (k0 + KB - 1 > qw) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + b * 32 + 8 * (i >> 2) + 4 * h + (i & 3) > qrow) s[b][i] = -INFINITY;
    }
    float tm = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) tm = fmaxf(tm, s[b][i]);
    tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
    const float m_new = fmaxf(m, tm);
    const float alpha = __builtin_amdgcn_exp2f((m - m_new) * a.c);
    const float mc = m_new * a.c;
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] *= alpha;
    u32x4 pf[4];   // [16-key group][two keys a register]
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][i], a.c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], a.c, -mc));
        l += p0 + p1;
        pf[b * 2 + (i >> 3)][(i & 7) >> 1] = cvt2<T>(p0, p1);
      }
    const int vr = 4 * h + ((lane & 15) >> 2);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v8 p8 = __builtin_bit_cast(v8, pf[g]);
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) {
        const int ch = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        const int key = g * 16 + vr;
        const u32x2 v0 = lds_tr16<T>(sV + key * ROWB + (swz_v<HD>(key, ch) << 4) + (lane & 1) * 8);
        const u32x2 v1 = lds_tr16<T>(sV + (key + 8) * ROWB + (swz_v<HD>(key + 8, ch) << 4) + (lane & 1) * 8);
        o[dt] = Mma<T>::m32(join8<T>(v0, v1), p8, o[dt]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (qrow >= len) return;
  const float inv = 1.0f / l;
  T* op = (T*)a.o + (size_t)(seq + qrow) * a.o_ts + (size_t)head * a.o_hs;
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      u32x2 st = {cvt2<T>(o[dt][i] * inv, o[dt][i + 1] * inv), cvt2<T>(o[dt][i + 2] * inv, o[dt][i + 3] * inv)};
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
  std::sort(w, w + at, [bm](const int4& x, const int4& y) {
    const int kx = std::min(x.z + bm, x.y), ky = std::min(y.z + bm, y.y);
    return kx != ky ? kx > ky : x.x != y.x ? x.x < y.x : x.z < y.z;
  });
  return at;
}

extern "C" int orc_attn_tile(const int32_t* lens, int n, int n_heads) {
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
