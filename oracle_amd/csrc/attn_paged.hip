// Decode attention over the paged KV cache for a batch whose rows share a long prefix (orc_kv_attend), grouped heads, bf16 / fp16.
//
// out[i] = sum_j p_j v_j / sum_j p_j over the first limits[i] tokens of row rows[i], p_j = exp2(c (q_i . k_j - m)), c = scale * log2(e).
// The sum is split: the shared prefix is read once for ALL queries of the batch (they are the columns of one matrix product per K/V head),
// every row's own tokens are read for its n_heads / n_kv_heads query heads. Each part leaves (m, sum, unnormalised output) in fp32;
// combine_kernel joins the parts of a query by exp2(c (m_part - m)).
//
// A workgroup = 4 waves that share 16 QT query columns and split the keys: every wave streams tiles of 32 keys of its own through a 2-deep
// LDS ring (LDS-DMA, no barrier in the loop), so the loop waits for memory only. Orientation as in attn.hip: S^T = K . Q^T, then
// O^T = V^T . P^T with the lane's own probabilities as the B operand and V^T by the transposing LDS read.
#include "../../include/oracle_hip.h"
#include "kernels.h"
#include "mma16.h"

namespace {

constexpr int KT = 32;            // keys of a wave's tile
constexpr int MAX_PARTS = 64;     // parts of one query (a lane of the combining wave each)

struct AttendArgs {
  const char *k, *v;              // this layer's K / V pages
  long page_elems;
  const int *table, *lens, *rows, *limits;
  int* status;
  const char* q; char* o;
  long q_ts, q_hs, o_ts, o_hs;
  float *ml, *po;                 // parts: [query][head][part] (m, sum), and the output sums
  int n_pages, log_ps, hkv, group, hq, max_rows, width, n, prefix, mt, gt, sp, ss;
  float c;
};

template <int HD> __device__ __forceinline__ int swz_k(int key, int ch) { return HD == 128 ? ch ^ (key & 15) : ch ^ ((key >> 1) & 7); }
template <int HD> __device__ __forceinline__ int swz_v(int key, int ch) {
  return HD == 128 ? ch ^ ((key & 7) << 1) : ch ^ (((key >> 1) & 3) << 1);
}

// tokens of row rows[i] that query i reads; *row: that row, -1 where it is outside the table
__device__ __forceinline__ int visible(const AttendArgs& a, int i, int* row) {
  const int r = a.rows[i];
  *row = r >= 0 && r < a.max_rows ? r : -1;
  if (*row < 0) return 0;
  int lim = a.lens[r];
  if (a.limits && a.limits[i] < lim) lim = a.limits[i];
  const int cap = a.width << a.log_ps;
  return lim < 0 ? 0 : lim > cap ? cap : lim;
}

// the first named row that holds the whole prefix (rows[0] where none does), by one wave
__device__ __forceinline__ int prefix_row(const AttendArgs& a, int lane) {
  for (int base = 0; base < a.n; base += 64) {
    const int i = base + lane;
    int r = -1;
    if (i < a.n) {
      r = a.rows[i];
      if (r < 0 || r >= a.max_rows || a.lens[r] < a.prefix) r = -1;
    }
    const unsigned long long hit = __ballot(r >= 0);
    if (hit) return __builtin_amdgcn_readlane(r, __builtin_ctzll(hit));
  }
  const int r = a.rows[0];
  return r >= 0 && r < a.max_rows ? r : -1;
}

template <typename T, int HD, int QT>
__global__ __launch_bounds__(256, 1) void attend_kernel(AttendArgs a) {
  typedef typename Mma<T>::v8 v8;
  constexpr int ROWB = HD * 2, CH = HD / 8, TILE = KT * ROWB, STAGE = 2 * TILE, RND = TILE / 1024, KPR = 64 / CH, MT = 16 * QT;
  constexpr int RING = 4 * 2 * STAGE, JOIN = (8 * MT + 4 * MT * HD) * 4;
  __shared__ __attribute__((aligned(16))) char smem[RING > JOIN ? RING : JOIN];   // 4 waves x 2 stages x (K | V); afterwards the waves' sums
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  const int ps = 1 << a.log_ps, n_pre = a.hkv * a.mt * a.sp;
  int kvh, part, k_lo, k_hi, row, f0;   // f0: first of the item's query columns; a column is (query, head of the group)
  int cols;
  const bool pre = (int)blockIdx.x < n_pre;
  if (pre) {
    const int pairs = a.hkv * a.sp, pair = blockIdx.x % pairs, mt = blockIdx.x / pairs;   // column tiles of one key range: one XCD where pairs % 8 == 0
    kvh = pair % a.hkv;
    part = pair / a.hkv;
    const int per = ((a.prefix + KT - 1) / KT + a.sp - 1) / a.sp * KT;
    k_lo = part * per;
    k_hi = k_lo + per < a.prefix ? k_lo + per : a.prefix;
    row = prefix_row(a, lane);
    f0 = mt * MT;
    cols = a.n * a.group - f0;
  } else {
    int x = blockIdx.x - n_pre;
    kvh = x % a.hkv; x /= a.hkv;
    const int gt = x % a.gt; x /= a.gt;
    const int sx = x % a.ss, i = x / a.ss;
    const int lim = visible(a, i, &row);
    if (a.prefix && kvh == 0 && gt == 0 && sx == 0 && w == 0 && row >= 0) {   // what it reads as shared, is it the same pages?
      const int pr = prefix_row(a, lane), held = ((lim < a.prefix ? lim : a.prefix) + ps - 1) >> a.log_ps;
      bool differ = false;
      for (int j = lane; j < held; j += 64) differ |= pr < 0 || a.table[(size_t)row * a.width + j] != a.table[(size_t)pr * a.width + j];
      if (__any(differ) && lane == 0) atomicOr(a.status, (int)ORC_KV_NOT_SHARED);
    }
    const int tiles = (lim - a.prefix + KT - 1) / KT;
    int per = (tiles + a.ss - 1) / a.ss;
    per = (per < 4 ? 4 : per) * KT;   // at least a tile for each wave
    k_lo = a.prefix + sx * per;
    k_hi = k_lo + per < lim ? k_lo + per : lim;
    part = a.sp + sx;
    f0 = i * a.group + gt * MT;
    cols = a.group - gt * MT;
  }
  if (cols > MT) cols = MT;
  const int nq = (cols + 15) >> 4;

  // the lane's query columns: c16 of every block of 16
  int lim_c[QT];
  v8 qf[QT][HD / 32];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int col = t * 16 + c16;
    lim_c[t] = 0;
    const int f = f0 + (col < cols ? col : 0), i = f / a.group, head = kvh * a.group + f % a.group;
    if (col < cols) {
      int r;
      const int lim = visible(a, i, &r);
      lim_c[t] = lim < k_hi ? lim : k_hi;
    }
    const T* qp = (const T*)a.q + (size_t)i * a.q_ts + (size_t)head * a.q_hs + g * 8;
#pragma unroll
    for (int kk = 0; kk < HD / 32; ++kk) qf[t][kk] = *(const v8*)(qp + kk * 32);
  }

  const T* kb = (const T*)a.k + (size_t)kvh * ps * HD;
  const T* vb = (const T*)a.v + (size_t)kvh * ps * HD;
  char* ring = smem + w * 2 * STAGE;
  const int key_p = lane / CH, ch_p = lane % CH;
  // Pages of a tile's two halves of 16 keys. A page outside the pool: the half is not attended, and its lanes load a token of the other half.
  auto page_of = [&](int k0) {
    int p = -1;
    if (row >= 0 && k0 < k_hi) p = a.table[(size_t)row * a.width + (k0 >> a.log_ps)];
    p = __builtin_amdgcn_readfirstlane(p);
    return p < a.n_pages ? p : -1;
  };
  auto dma = [&](int k0, int p0, int p1, int stage) {
    char* sk = ring + stage * STAGE;
    const int last = k_hi - 1;
#pragma unroll
    for (int r = 0; r < RND; ++r) {
      const int key = r * KPR + key_p;
      int at = k0 + key, page = key < 16 ? p0 : p1;
      if (page < 0) { page = key < 16 ? p1 : p0; at = key < 16 ? k0 + 16 : k0; }
      if (at > last) { at = last; page = (last - k0) < 16 ? p0 : p1; if (page < 0) { page = p0; at = k0; } }
      const size_t off = (size_t)page * a.page_elems + (size_t)(at & (ps - 1)) * HD;
      __builtin_amdgcn_global_load_lds((glb_void_t*)(kb + off + swz_k<HD>(key, ch_p) * 8), (lds_void_t*)(sk + r * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_void_t*)(vb + off + swz_v<HD>(key, ch_p) * 8), (lds_void_t*)(sk + TILE + r * 1024), 16, 0, 0);
    }
  };

  f32x4 o[QT][HD / 16];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // tiles w, w + 4, ... of the range; a tile none of whose pages is in the pool is passed over
  int k0 = k_lo + w * KT, p0 = -1, p1 = -1;
  auto seek = [&](int from) {
    for (; from < k_hi; from += 4 * KT) {
      p0 = page_of(from);
      p1 = page_of(from + 16);
      if (p0 >= 0 || p1 >= 0) break;
    }
    return from;
  };
  k0 = seek(k0);
  if (k0 < k_hi) dma(k0, p0, p1, 0);
  int stage = 0;
  while (k0 < k_hi) {
    const bool ok0 = p0 >= 0, ok1 = p1 >= 0;
    const int nx = seek(k0 + 4 * KT);
    if (nx < k_hi) {
      dma(nx, p0, p1, stage ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * RND) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const char* sK = ring + stage * STAGE;
    const char* sV = sK + TILE;
    f32x4 s[QT][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int key = b * 16 + c16;
#pragma unroll
      for (int kk = 0; kk < HD / 32; ++kk) {
        const v8 kf = *(const v8*)(sK + key * ROWB + (swz_k<HD>(key, kk * 4 + g) << 4));
#pragma unroll
        for (int t = 0; t < QT; ++t)
          if (t < nq) s[t][b] = Mma<T>::m16(kf, qf[t][kk], s[t][b]);
      }
    }
    v8 pf[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      if (t >= nq) continue;
      float tm = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool see = k0 + b * 16 + 4 * g + r < lim_c[t] && (b ? ok1 : ok0);
          s[t][b][r] = see ? s[t][b][r] : -INFINITY;
          tm = fmaxf(tm, s[t][b][r]);
        }
      tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
      tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
      const float m_new = fmaxf(m[t], tm), mu = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m[t] - mu) * a.c);
      m[t] = m_new;
      l[t] *= alpha;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[t][d] *= alpha;
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f((s[t][j >> 2][j & 3] - mu) * a.c);
        l[t] += p[j];
      }
      pf[t] = __builtin_bit_cast(v8, (u32x4){cvt2<T>(p[0], p[1]), cvt2<T>(p[2], p[3]), cvt2<T>(p[4], p[5]), cvt2<T>(p[6], p[7])});
    }
    const int key = 4 * g + (c16 >> 2);
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      const int ch = d * 2 + ((lane & 3) >> 1);
      const u32x2 v0 = lds_tr16<T>(sV + key * ROWB + (swz_v<HD>(key, ch) << 4) + (lane & 1) * 8);
      const u32x2 v1 = lds_tr16<T>(sV + (key + 16) * ROWB + (swz_v<HD>(key + 16, ch) << 4) + (lane & 1) * 8);
      const v8 vf = join8<T>(v0, v1);
#pragma unroll
      for (int t = 0; t < QT; ++t)
        if (t < nq) o[t][d] = Mma<T>::m16(vf, pf[t], o[t][d]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this stage's reads are done before the next pass's DMA goes into it
    stage ^= 1;
    k0 = nx;
  }

  // join the four waves
  __syncthreads();
  float* sm = (float*)smem;                  // [4][MT] maxima, [4][MT] sums, then [4][MT][HD]
  float* so = sm + 8 * MT;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    l[t] += __shfl_xor(l[t], 16, 64);
    l[t] += __shfl_xor(l[t], 32, 64);
    if (g == 0) { sm[w * MT + t * 16 + c16] = m[t]; sm[(4 + w) * MT + t * 16 + c16] = l[t]; }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int col = t * 16 + c16;
    float mx = -INFINITY;
    for (int x = 0; x < 4; ++x) mx = fmaxf(mx, sm[x * MT + col]);
    const float f = m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[t] - mx) * a.c);
    const bool any = l[t] != 0.f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
      *(f32x4*)(so + ((size_t)w * MT + col) * HD + d * 16 + 4 * g) = any ? o[t][d] * f : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  const int parts = a.sp + a.ss;
  for (int x = threadIdx.x; x < cols * (HD / 4); x += 256) {
    const int col = x / (HD / 4), d4 = x % (HD / 4);
    float mx = -INFINITY, sum = 0.f;
    for (int y = 0; y < 4; ++y) mx = fmaxf(mx, sm[y * MT + col]);
    for (int y = 0; y < 4; ++y) {
      const float my = sm[y * MT + col], ly = sm[(4 + y) * MT + col];
      if (ly != 0.f) sum += ly * __builtin_amdgcn_exp2f((my - mx) * a.c);
    }
    f32x4 v = *(const f32x4*)(so + (size_t)col * HD + d4 * 4);
    for (int y = 1; y < 4; ++y) v += *(const f32x4*)(so + ((size_t)y * MT + col) * HD + d4 * 4);
    const int f = f0 + col, i = f / a.group, head = kvh * a.group + f % a.group;
    if (parts == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      u32x2 st = {cvt2<T>(v[0] * inv, v[1] * inv), cvt2<T>(v[2] * inv, v[3] * inv)};
      *(u32x2*)((T*)a.o + (size_t)i * a.o_ts + (size_t)head * a.o_hs + d4 * 4) = st;
    } else {
      const size_t at = ((size_t)i * a.hq + head) * parts + part;
      if (d4 == 0) { a.ml[2 * at] = mx; a.ml[2 * at + 1] = sum; }
      if (sum != 0.f) *(f32x4*)(a.po + at * HD + d4 * 4) = v;
    }
  }
}

// one wave per (query, head): lane s holds part s
template <typename T, int HD>
__global__ __launch_bounds__(256) void combine_kernel(AttendArgs a) {
  const int lane = threadIdx.x & 63;
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= (long)a.n * a.hq) return;
  const int parts = a.sp + a.ss;
  float m = -INFINITY, l = 0.f;
  if (lane < parts) { m = a.ml[2 * (id * parts + lane)]; l = a.ml[2 * (id * parts + lane) + 1]; }
  if (l == 0.f) m = -INFINITY;
  const float mx = wave_max(m);
  const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - mx) * a.c);
  const float sum = wave_sum(l * f);
  float acc[HD / 64];
#pragma unroll
  for (int d = 0; d < HD / 64; ++d) acc[d] = 0.f;
  for (int s = 0; s < parts; ++s) {
    if (__shfl(l, s, 64) == 0.f) continue;
    const float fs = __shfl(f, s, 64);
    const float* po = a.po + (id * parts + s) * HD + lane * (HD / 64);
#pragma unroll
    for (int d = 0; d < HD / 64; ++d) acc[d] = fmaf(po[d], fs, acc[d]);
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int i = (int)(id / a.hq), head = (int)(id % a.hq);
  T* op = (T*)a.o + (size_t)i * a.o_ts + (size_t)head * a.o_hs + lane * (HD / 64);
  if constexpr (HD == 128) *(uint32_t*)op = cvt2<T>(acc[0] * inv, acc[1] * inv);
  else *op = (T)(acc[0] * inv);
}

// how a call is split; the same for the scratch size and the launch
struct Split { int qt, mt, gt, sp, ss; };
Split split_of(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  Split s;
  const int group = n_heads / c->n_kv_heads;
  const int64_t cols = (int64_t)n * group;
  const int64_t most = prefix ? cols : group;
  s.qt = most <= 16 ? 1 : most <= 32 ? 2 : 4;
  s.mt = prefix ? (int)((cols + 16 * s.qt - 1) / (16 * s.qt)) : 0;
  s.gt = (group + 16 * s.qt - 1) / (16 * s.qt);
  s.sp = 0;
  if (prefix) {
    const int64_t base = (int64_t)c->n_kv_heads * s.mt;
    int64_t sp = (512 + base - 1) / base;
    const int64_t most_sp = (prefix + 255) / 256;
    sp = sp < most_sp ? sp : most_sp;
    s.sp = (int)(sp < 1 ? 1 : sp > 32 ? 32 : sp);
  }
  const int64_t own = (int64_t)n * c->n_kv_heads * s.gt;
  const int64_t left = (int64_t)c->max_row_pages * c->page_size - prefix;
  int64_t ss = (512 + own - 1) / own;
  const int64_t most_ss = (left + 255) / 256;
  ss = ss < most_ss ? ss : most_ss;
  s.ss = (int)(ss < 1 ? 1 : ss > 16 ? 16 : ss);
  return s;
}

const char* bad_call(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  if (!c) return "null argument";
  if (c->n_kv_heads < 1 || n_heads < 1 || n_heads % c->n_kv_heads) return "n_heads is not a multiple of n_kv_heads";
  if (n < 0 || n > 1024) return "0..1024 queries a call";
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return "page_size is 16, 32, 64 or 128";
  if (c->max_rows < 1 || c->n_pages < 1 || c->max_row_pages < 1 || c->max_row_pages > 1 << 20) return "bad geometry";
  if (prefix < 0 || prefix % c->page_size || (int64_t)prefix > (int64_t)c->max_row_pages * c->page_size)
    return "prefix_tokens is not a multiple of page_size inside a row";
  return nullptr;
}

template <typename T, int HD, int QT> hipError_t launch_qt(const AttendArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)(a.hkv * a.mt * a.sp + a.n * a.hkv * a.gt * a.ss);
  hipLaunchKernelGGL((attend_kernel<T, HD, QT>), dim3(grid), dim3(256), 0, s, a);
  if (a.sp + a.ss > 1)
    hipLaunchKernelGGL((combine_kernel<T, HD>), dim3((unsigned)(((int64_t)a.n * a.hq + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename T, int HD> hipError_t launch_hd(const AttendArgs& a, int qt, hipStream_t s) {
  return qt == 1 ? launch_qt<T, HD, 1>(a, s) : qt == 2 ? launch_qt<T, HD, 2>(a, s) : launch_qt<T, HD, 4>(a, s);
}

}  // namespace

extern "C" int64_t orc_kv_attend_ws(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  const char* bad = bad_call(c, n, n_heads, prefix);
  if (bad) return orc_fail("orc_kv_attend_ws", bad);
  const Split s = split_of(c, n < 1 ? 1 : n, n_heads, prefix);
  return s.sp + s.ss == 1 ? 0 : (int64_t)n * n_heads * (s.sp + s.ss) * (c->head_dim + 2) * 4;
}

extern "C" int orc_kv_attend(const orc_kv_pages* c, int layer, const void* q, void* out, const int64_t* st, const int32_t* rows,
                             const int32_t* limits, int n, int n_heads, int prefix, float scale, void* ws, void* stream) {
  const char* who = "orc_kv_attend";
  const char* bad = bad_call(c, n, n_heads, prefix);
  if (bad) return orc_fail(who, bad);
  if (c->head_dim != 64 && c->head_dim != 128) return orc_fail(who, "head_dim is 64 or 128");
  if (c->dtype != 0 && c->dtype != 1) return orc_fail(who, "dtype is 0 (bf16) or 1 (fp16)");
  if (layer < 0 || layer >= c->n_layers) return orc_fail(who, "layer outside the cache");
  if (!(scale > 0.f) || !(scale < 1e30f)) return orc_fail(who, "scale is not positive and finite");
  if (!st) return orc_fail(who, "null argument");
  for (int i = 0; i < 4; ++i)
    if (st[i] < 0 || st[i] % 8) return orc_fail(who, "strides are not multiples of 8 elements");
  if (n == 0) return 0;
  const Split s = split_of(c, n, n_heads, prefix);
  if (!q || !out || !rows || !c->kv || !c->table || !c->lens || !c->status || (s.sp + s.ss > 1 && !ws)) return orc_fail(who, "null argument");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)c->kv | (uintptr_t)ws) & 15) return orc_fail(who, "tensors are not aligned to 16 bytes");
  AttendArgs a;
  const size_t page = (size_t)c->n_kv_heads * c->page_size * c->head_dim;
  a.k = (const char*)c->kv + (size_t)layer * 2 * c->n_pages * page * 2;
  a.v = a.k + (size_t)c->n_pages * page * 2;
  a.page_elems = (long)page;
  a.table = c->table; a.lens = c->lens; a.rows = rows; a.limits = limits; a.status = c->status;
  a.q = (const char*)q; a.o = (char*)out;
  a.q_ts = st[0]; a.q_hs = st[1]; a.o_ts = st[2]; a.o_hs = st[3];
  const int64_t parts = (int64_t)n * n_heads * (s.sp + s.ss);
  a.po = (float*)ws; a.ml = (float*)ws + parts * c->head_dim;
  a.n_pages = c->n_pages; a.log_ps = __builtin_ctz(c->page_size); a.hkv = c->n_kv_heads; a.group = n_heads / c->n_kv_heads; a.hq = n_heads;
  a.max_rows = c->max_rows; a.width = c->max_row_pages; a.n = n; a.prefix = prefix; a.mt = s.mt; a.gt = s.gt; a.sp = s.sp; a.ss = s.ss;
  a.c = scale * 1.4426950408889634f;
  hipStream_t hs = (hipStream_t)stream;
  hipError_t e;
  if (c->dtype == 0) e = c->head_dim == 128 ? launch_hd<__bf16, 128>(a, s.qt, hs) : launch_hd<__bf16, 64>(a, s.qt, hs);
  else e = c->head_dim == 128 ? launch_hd<_Float16, 128>(a, s.qt, hs) : launch_hd<_Float16, 64>(a, s.qt, hs);
  return e == hipSuccess ? 0 : orc_fail(who, hipGetErrorString(e));
}
