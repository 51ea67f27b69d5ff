// Decode attention over the paged KV cache for a batch whose rows share a long prefix (orc_kv_attend), grouped heads, bf16 / fp16.
//
// out[i] = sum_j p_j v_j / sum_j p_j over the first limits[i] tokens of row rows[i], p_j = exp2(c (q_i . k_j - m)), c = scale * log2(e).
// The sum is split: the shared prefix is read once for ALL queries of the batch (they are the columns of one matrix product per K/V head),
// every row's own tokens are read for its n_heads / n_kv_heads query heads. Each part leaves (m, sum, unnormalised output) in fp32;
// combine_kernel joins the parts of a query by exp2(c (m_part - m)): a launch of its own, 4 us after 19 us of attention for 16 rows over 2304 shared
// tokens. (The last workgroup of a query could do it; that takes counters cleared before the call and a write-back of every XCD's L2.)
//
// Two shapes of work, 4 waves each:
//   keys_item  16 query columns (one row's heads over its own tokens, or a small batch over the prefix): the waves share the columns and
//              split the keys. A wave's tile is 32 keys, K straight to registers in operand order, V through 8 KiB of LDS of its own; no
//              barrier in the loop and little LDS, so 4 workgroups fit a CU and hide each other's memory latency. Bound by latency: 16 rows of 32 heads, 2304
//              shared and up to 300 own tokens, 66 MB in 18.6 us (3.6 TB/s, out of the Infinity Cache where calls follow one another), 7 of
//              them with hardly a byte to read (launch, lengths, page ids, first tile); over 12 layers in turn, which that cache does not hold, the call
//              takes 26.7 us instead of 23.0.
//   cols_item  many columns over the prefix: every wave has 32 columns of its own, 64-key tiles go through a 2-deep LDS ring that
//              the waves share (flash32.h). Bound by the matrix cores and the softmax between the two products, then by the rows' own tokens: 96 rows of 32
//              heads on 8, 32k shared and up to 2000 own tokens, 108 us = 490 TFLOP/s and 3.3 TB/s at once (the prefix's items first: own
//              ones put first or between them were up to twice as slow, the workgroups being dealt out in turn). A query that ends inside the prefix
//              sends every item up to whose end it does not reach to keys_item, 16 columns at a time: 96 rows with own tokens spread evenly
//              over 0..2000 127 -> 318 us where one of them ends 100 tokens before the prefix does, 368 where it ends at 16000.
// The rows' own tokens are cut by the sizes that the host knows (split_of), not by their lengths: MAX_SS parts a row at the most, one from 512 (row, K/V
// head) pairs on. A batch with one row far longer than the others waits for it: 64 rows of 100 tokens and one of 32k, 8 K/V heads, 427 us (its bytes take
// 32); one row of 32k alone, 1 / 2 / 8 / 32 K/V heads, 32 / 35 / 37 / 100 us (bytes 3 / 7 / 26 / 105).
// The page ids of an item's keys are gathered into LDS first, so that the loop's addresses wait for no dependent load.
#include <type_traits>

#include "../../include/oracle_hip.h"
#include "flash32.h"
#include "kernels.h"

namespace {

constexpr int KT = 32;            // keys of a wave's tile in keys_item
constexpr int IDS = 512;          // page ids held in LDS at a time by keys_item
constexpr int IDS_COLS = 2048;    // by cols_item, whose range has to fit
constexpr int MAX_SP = 40, MAX_SS = 16;   // parts of a query, of the prefix and of its row's own tokens
constexpr int UNIT_COLS = 64, UNIT_KEYS = KT;   // keys of a tile: parts of the prefix are whole ones
static_assert(UNIT_COLS == Tile64<64>::KEYS && UNIT_COLS == Tile64<128>::KEYS);
static_assert(MAX_SP + MAX_SS <= 64, "a lane of the combining wave each");

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

// places of the 16-byte chunks of a V row in keys_item's tile: the 8 keys x 32 bytes of half a transposing read fall on different banks
template <int HD> __device__ __forceinline__ int swz_v16(int key, int ch) {
  return HD == 128 ? ch ^ ((key & 7) << 1) : ch ^ (((key >> 1) & 3) << 1);
}

// tokens of row rows[i] that query i reads; *row: that row, -1 where it is outside the table. No branch, so that other loads need not wait.
__device__ __forceinline__ int visible(const AttendArgs& a, int i, int* row) {
  const int r = a.rows[i], cap = a.width << a.log_ps;
  const bool ok = r >= 0 && r < a.max_rows;
  int lim = a.lens[ok ? r : 0];
  const int most = a.limits ? a.limits[i] : cap;
  lim = most < lim ? most : lim;
  lim = lim < cap ? lim : cap;
  *row = ok ? r : -1;
  return ok && lim > 0 ? lim : 0;
}

// Whether query i has any token to attend, where the sum over its keys came out as 0 (rare: a row without tokens). If it has, all its scores are -inf,
// and the softmax is 0 / 0.
__device__ bool attends(const AttendArgs& a, int i) {
  int r;
  const int lim = visible(a, i, &r);
  for (int j = 0; j << a.log_ps < lim; ++j) {
    const int page = a.table[(size_t)r * a.width + j];
    if (page >= 0 && page < a.n_pages) return true;
  }
  return false;
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

// What a workgroup does: the keys [k_lo, k_hi) of row `row` for `cols` query columns of K/V head kvh, from column f0 (query, head of the group) on
struct Item { int kvh, part, k_lo, k_hi, row, f0, cols; };

// ids[e] = page of the tokens [(first + e) ps, ...) of the row, -1 outside the pool; by the whole workgroup. Returns whether any is outside,
// or `odd` is set in any thread.
__device__ __forceinline__ bool load_ids(const AttendArgs& a, int row, int first, int count, int* ids, bool odd = false) {
  __syncthreads();
  for (int e = threadIdx.x; e < count; e += 256) {
    int p = row < 0 ? -1 : a.table[(size_t)row * a.width + first + e];
    p = p < a.n_pages ? p : -1;
    ids[e] = p;
    odd |= p < 0;
  }
  return __syncthreads_or(odd);
}

// One part of one column's result: m, sum and the output sums of dims d..d+3 (want_ml: by the caller that holds d == 0); the result itself where the
// column has no other part.
template <typename T, int HD>
__device__ __forceinline__ void put(const AttendArgs& a, const Item& it, int col, int d, float m, float sum, f32x4 v) {
  const int f = it.f0 + col, i = f / a.group, head = it.kvh * a.group + f % a.group;
  if (a.sp + a.ss == 1) {
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    u32x2 st = {cvt2<T>(v[0] * inv, v[1] * inv), cvt2<T>(v[2] * inv, v[3] * inv)};
    if (sum == 0.f) st[0] = st[1] = attends(a, i) ? cvt2<T>(NAN, NAN) : 0;
    *(u32x2*)((T*)a.o + (size_t)i * a.o_ts + (size_t)head * a.o_hs + d) = st;
  } else {
    const size_t at = ((size_t)i * a.hq + head) * (a.sp + a.ss) + it.part;
    if (d == 0) { a.ml[2 * at] = m; a.ml[2 * at + 1] = sum; }
    if (sum != 0.f) *(f32x4*)(a.po + at * HD + d) = v;
  }
}

// LDS of keys_item: a V tile for each wave and, behind the loop, its outputs, in the wave's own room. step: the rooms' distance in
// one array (picking a room by address arithmetic takes fewer registers, and 128 are the limit), 0 where they are arrays of their own.
struct Rooms { char* r[4]; int step; };

// Up to 16 columns. True where a value that some column does not see may have spoilt an output (it is infinite or NaN, and 0 times it is not 0).
template <typename T, int HD, int NID>
__device__ __forceinline__ bool keys_item(const AttendArgs& a, const Item& it, const Rooms& room, int* ids, float* sm) {
  typedef typename Mma<T>::v8 v8;
  constexpr int ROWB = HD * 2, CH = HD / 8, TILE = KT * ROWB, RND = TILE / 1024, KPR = 64 / CH;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));   // what follows from it is computed here, not held in registers around the loop of keys_items
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c16 = lane & 15;
  const int ps = 1 << a.log_ps;
  int lim;                        // of the lane's query column c16
  bool part;
  v8 qf[HD / 32];
  {
    const int f = it.f0 + (c16 < it.cols ? c16 : 0), i = f / a.group, head = it.kvh * a.group + f % a.group;
    int r;
    lim = visible(a, i, &r);
    lim = c16 < it.cols ? (lim < it.k_hi ? lim : it.k_hi) : 0;
    part = __any(lim > it.k_lo && lim < it.k_hi);   // (the waves hold the same columns)
    const T* qp = (const T*)a.q + (size_t)i * a.q_ts + (size_t)head * a.q_hs + g * 8;
#pragma unroll
    for (int kk = 0; kk < HD / 32; ++kk) qf[kk] = *(const v8*)(qp + kk * 32);
  }
  f32x4 o[HD / 16];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const size_t head_off = (size_t)it.kvh * ps * ROWB, page_bytes = (size_t)a.page_elems * 2;
  char* sV = room.step ? room.r[0] + w * room.step : w == 0 ? room.r[0] : w == 1 ? room.r[1] : w == 2 ? room.r[2] : room.r[3];
  const int key_p = lane / CH, ch_p = lane % CH;
  for (int kc = it.k_lo; kc < it.k_hi; kc += (NID - 2) << a.log_ps) {
    const int first = kc >> a.log_ps, ke = kc + ((NID - 2) << a.log_ps) < it.k_hi ? kc + ((NID - 2) << a.log_ps) : it.k_hi;
    load_ids(a, it.row, first, ((ke - 1) >> a.log_ps) - first + 1, ids);
    for (int k0 = kc + w * KT; k0 < ke; k0 += 4 * KT) {
      // The tile's two halves of 16 keys, each on one page. The buffer descriptors end with the last token (at once, for a page outside the pool), so
      // that what is not there arrives as zeros: its score is masked, and its value must not be something that 0 times it is not 0.
      const bool two = k0 + 16 < ke;
      const int p0 = __builtin_amdgcn_readfirstlane(ids[(k0 >> a.log_ps) - first]);
      const int p1 = two ? __builtin_amdgcn_readfirstlane(ids[((k0 + 16) >> a.log_ps) - first]) : -1;
      if (p0 < 0 && p1 < 0) continue;
      size_t off[2];
      int at[2], bytes[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int k = k0 + 16 * b, page = b ? p1 : p0;
        at[b] = (k & (ps - 1)) * ROWB;
        bytes[b] = page < 0 ? 0 : at[b] + (ke - k < 16 ? ke - k : 16) * ROWB;
        off[b] = (size_t)(page < 0 ? 0 : page) * page_bytes + head_off;
      }
      v8 kf[2][HD / 32];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk)
          kf[b][kk] = __builtin_bit_cast(v8, buffer_load16(buffer_of(a.k + off[b], bytes[b]), at[b] + c16 * ROWB + g * 16 + kk * 64));
#pragma unroll
      for (int r = 0; r < RND; ++r) {
        const int key = r * KPR + key_p, b = r / (RND / 2);
        buffer_load16_lds(buffer_of(a.v + off[b], bytes[b]), at[b] + (key - 16 * b) * ROWB + swz_v16<HD>(key, ch_p) * 16, sV + r * 1024);
      }
      f32x4 s[2];
      float tm = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) s[b] = Mma<T>::m16(kf[b][kk], qf[kk], s[b]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool see = k0 + b * 16 + 4 * g + r < lim && (b ? p1 : p0) >= 0;
          s[b][r] = see ? s[b][r] : -INFINITY;
          tm = fmaxf(tm, s[b][r]);
        }
      }
      tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
      tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
      const float m_new = fmaxf(m, tm), mu = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m - mu) * a.c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d] *= alpha;
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f((s[j >> 2][j & 3] - mu) * a.c);
        l += p[j];
      }
      u32x4 pw = {cvt2<T>(p[0], p[1]), cvt2<T>(p[2], p[3]), cvt2<T>(p[4], p[5]), cvt2<T>(p[6], p[7])};
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(pw)::"memory");   // V is in LDS. (With pw: otherwise the wait may move in front of the scores.)
      const v8 pf = __builtin_bit_cast(v8, pw);
      const int key = 4 * g + (c16 >> 2);
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        const int ch = d * 2 + ((lane & 3) >> 1);
        const u32x2 v0 = lds_tr16<T>(sV + key * ROWB + (swz_v16<HD>(key, ch) << 4) + (lane & 1) * 8);
        const u32x2 v1 = lds_tr16<T>(sV + (key + 16) * ROWB + (swz_v16<HD>(key + 16, ch) << 4) + (lane & 1) * 8);
        o[d] = Mma<T>::m16(join8<T>(v0, v1), pf, o[d]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the tile's reads are done before the next tile's DMA
    }
  }

  // Join the four waves: each leaves its maxima, sums and outputs (in its own room, 16-byte pieces permuted against bank conflicts); behind one
  // barrier every thread adds up its pieces of the columns.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) { sm[w * 16 + c16] = m; sm[(4 + w) * 16 + c16] = l; }
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) *(f32x4*)(sV + c16 * HD * 4 + (((d * 4 + g) ^ c16) << 4)) = o[d];
  __syncthreads();
  bool odd = false;
  for (int x = tid; x < it.cols * (HD / 4); x += 256) {
    const int col = x / (HD / 4), d4 = x % (HD / 4);
    float mx = -INFINITY, sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < 4; ++y) mx = fmaxf(mx, sm[y * 16 + col]);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float ly = sm[(4 + y) * 16 + col], f = __builtin_amdgcn_exp2f((sm[y * 16 + col] - mx) * a.c);
      if (ly != 0.f) {            // a wave without keys for this column: nothing to add (its maximum is -inf)
        sum += ly * f;
        v += *(const f32x4*)(room.r[y] + col * HD * 4 + ((d4 ^ col) << 4)) * f;
      }
    }
    put<T, HD>(a, it, col, d4 * 4, mx, sum, v);
    odd |= !(fmaf(v[0], 0.f, v[1] * 0.f) + fmaf(v[2], 0.f, v[3] * 0.f) == 0.f);
  }
  return part && __builtin_amdgcn_readfirstlane(__syncthreads_or(odd));   // a scalar: a loop around it stays one of the whole wave
}

// The item's columns, 16 at a time; where a value that not all of them see is infinite or NaN, again one by one, up to the column's last token.
// A barrier in front of every pass but the first: its waves write sm and the rooms, which the pass before still joins (with one column by a single
// wave), and a pass whose column ends in front of the item has no load_ids to wait in.
template <typename T, int HD, int NID>
__device__ __forceinline__ void keys_items(const AttendArgs& a, const Item& it, const Rooms& room, int* ids, float* sm) {
  Item sub = it;
  int x = 0, wide = 16, back = 0;
  for (bool first = true; x < it.cols; first = false) {
    if (!first) __syncthreads();
    sub.f0 = it.f0 + x;
    sub.cols = it.cols - x < wide ? it.cols - x : wide;
    sub.k_hi = it.k_hi;
    if (wide == 1) {
      int r;
      const int lim = visible(a, sub.f0 / a.group, &r);
      sub.k_hi = lim < it.k_hi ? lim : it.k_hi;
    }
    if (keys_item<T, HD, NID>(a, sub, room, ids, sm)) {
      back = x + sub.cols;
      wide = 1;
      continue;
    }
    x += sub.cols;
    if (x == back) wide = 16;
  }
}

// Where cols_item's tiles come from (flash_loop): the pages ids[] of the tokens [kc, ke), all of them in the pool. A lane holds where page win + lane
// starts, so that an address takes two v_readlanes and no LDS round trip; the window moves on once in a while.
template <typename T, int HD> struct PageSrc {
  typedef Tile64<HD> Tile;
  static constexpr int RND = Tile::KEYS * Tile::CH / 256, KPR = 256 / Tile::CH, GK = KPR / 4;   // GK: keys of one DMA instruction, all on one page
  const char *kb, *vb;
  const int* ids;
  unsigned page_bytes;
  int kc, ke, first, last, log_ps, w, h, lane, win;
  unsigned lk, lv, lo, hi;
  __device__ __forceinline__ void window(int at) {
    win = at;
    const unsigned long long off = (unsigned long long)(unsigned)ids[win + lane < IDS_COLS ? win + lane : IDS_COLS - 1] * page_bytes;
    lo = (unsigned)off;
    hi = (unsigned)(off >> 32);
  }
  __device__ __forceinline__ void init(int tid) {
    const int key_p = tid / Tile::CH;
    w = __builtin_amdgcn_readfirstlane(tid >> 6);
    lane = tid & 63;
    h = lane >> 5;
    first = kc >> log_ps;
    last = ((ke - 1) >> log_ps) - first;
    lk = (unsigned)((key_p - w * GK) * HD + Tile::swz_k(key_p, tid % Tile::CH) * 8) * 2;
    lv = (unsigned)((key_p - w * GK) * HD + Tile::swz_v(key_p, tid % Tile::CH) * 8) * 2;
    window(0);
  }
  __device__ __forceinline__ void next(int t) {   // K of tile t + 2 and V of t + 1 are to come: their pages are in the window
    const int k = (kc + (t + 3) * Tile::KEYS - 1) >> log_ps, v = (kc + (t + 1) * Tile::KEYS) >> log_ps;
    if (min(k - first, last) - win >= 64) window(min(v - first, last));
  }
  // The r-th DMA instruction of tile t; what lies behind the last token arrives as zeros (a descriptor of no bytes).
  __device__ __forceinline__ void ask(const char* base, unsigned l, int t, int r, char* to) const {
    const int k = kc + t * Tile::KEYS + r * KPR + w * GK, e = min((k >> log_ps) - first, last) - win;
    const unsigned long long off = (unsigned)__builtin_amdgcn_readlane((int)lo, e) | (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)hi, e) << 32;
    const char* from = base + off + (unsigned)(k & ((1 << log_ps) - 1)) * (HD * 2);
    buffer_load16_lds(buffer_of(from, k < ke ? GK * HD * 2 : 0), (int)l, to + w * 1024 + r * 4096);
  }
  __device__ __forceinline__ void K(int t, int r, char* to) const { ask(kb, lk, t, r, to); }
  __device__ __forceinline__ void V(int t, int r, char* to) const { ask(vb, lv, t, r, to); }
  __device__ __forceinline__ void mask_last(int t, f32x16 (&s)[2]) const {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kc + t * Tile::KEYS + Flash32<T, HD>::key_of(b, i, h) >= ke) s[b][i] = -INFINITY;
  }
};

// Up to 128 columns. False, and nothing done, where a page is outside the pool or a query ends before the item's keys do: keys_items has a test for
// every key.
template <typename T, int HD>
__device__ __forceinline__ bool cols_item(const AttendArgs& a, const Item& it, const Images& im, int* ids) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int ps = 1 << a.log_ps, col = w * 32 + (lane & 31);
  const int fc = it.f0 + (col < it.cols ? col : 0), i = fc / a.group;
  int r;
  const int lim = visible(a, i, &r);
  const bool empty = lim == 0;             // a column whose query has no tokens (a row that has ended): what it computes is not used
  const int first = it.k_lo >> a.log_ps;
  if (load_ids(a, it.row, first, ((it.k_hi - 1) >> a.log_ps) - first + 1, ids, lim > 0 && lim < it.k_hi)) return false;
  PageSrc<T, HD> src;
  src.kb = a.k + (size_t)it.kvh * ps * HD * 2;
  src.vb = a.v + (size_t)it.kvh * ps * HD * 2;
  src.ids = ids; src.page_bytes = (unsigned)(a.page_elems * 2); src.log_ps = a.log_ps;
  src.kc = it.k_lo; src.ke = it.k_hi;
  src.init(threadIdx.x);
  Flash32<T, HD> f;
  f.init((const T*)a.q + (size_t)i * a.q_ts + (size_t)(it.kvh * a.group + fc % a.group) * a.q_hs, lane);
  const int tiles = (it.k_hi - it.k_lo + Tile64<HD>::KEYS - 1) / Tile64<HD>::KEYS;
  flash_loop(f, src, im, tiles, w * 32 < it.cols ? tiles : 0, a.c);   // a wave without columns helps with the loads
  const float sum = empty ? 0.f : f.total();
  // (with a prefix there are two parts at least: never the result itself)
  const int at = (i * a.hq + it.kvh * a.group + fc % a.group) * (a.sp + a.ss) + it.part;
  if (col < it.cols && h == 0) { a.ml[2 * (size_t)at] = f.m; a.ml[2 * (size_t)at + 1] = sum; }
  f.template rows<true>(im.of(w), lane, 1.f, [&](int row, int byte, u32x4 v) {
    const int to = __shfl(at, row, 64);
    if (w * 32 + row < it.cols) *(u32x4*)((char*)(a.po + (size_t)to * HD) + byte) = v;
  });
  return true;
}

// COLS: the prefix is read by cols_item, 128 query columns at a time; else by keys_item, 16
template <typename T, int HD, bool COLS>
__global__ __launch_bounds__(256, COLS ? (HD == 64 ? 3 : 2) : 4) void attend_kernel(AttendArgs a) {
  constexpr int MT = COLS ? 128 : 16, NID = COLS ? IDS_COLS : IDS;
  // a room holds a V tile of 32 keys, or 16 columns' outputs (as much); the tile images of cols_item are larger
  constexpr int ROOM = COLS ? Tile64<HD>::BYTES : KT * HD * 2, ONE = COLS ? ROOM : 16;
  static_assert(16 * HD * 4 <= KT * HD * 2, "the outputs fit the V tile");
  __shared__ __attribute__((aligned(16))) char r0[COLS ? ROOM : 4 * ROOM], r1[ONE], r2[ONE], r3[ONE];
  const Rooms room = COLS ? Rooms{{r0, r1, r2, r3}, 0} : Rooms{{r0, r0 + ROOM, r0 + 2 * ROOM, r0 + 3 * ROOM}, ROOM};
  __shared__ int ids[NID];
  __shared__ float sm[8 * 16];           // the waves' maxima and sums
  const int lane = threadIdx.x & 63, pairs = a.hkv * a.sp, n_pre = pairs * a.mt;
  int x = (int)blockIdx.x - n_pre;
  Item it;
  if (x < 0) {
    const int p_at = blockIdx.x;
    int pair, mt;   // the column tiles of one key range behind one another and, where pairs divide by 8, on one XCD
    if ((pairs & 7) == 0) { pair = (p_at / 8 / a.mt) * 8 + (p_at & 7); mt = p_at / 8 % a.mt; }
    else { pair = p_at / a.mt; mt = p_at % a.mt; }
    it.kvh = pair % a.hkv;
    it.part = pair / a.hkv;
    constexpr int UNIT = COLS ? UNIT_COLS : UNIT_KEYS;
    const int per = ((a.prefix + UNIT - 1) / UNIT + a.sp - 1) / a.sp * UNIT;
    it.k_lo = it.part * per;
    it.k_hi = it.k_lo + per < a.prefix ? it.k_lo + per : a.prefix;
    it.row = prefix_row(a, lane);
    it.f0 = mt * MT;
    it.cols = a.n * a.group - it.f0;
    if (it.cols > MT) it.cols = MT;
    if constexpr (COLS)
      if (cols_item<T, HD>(a, it, Images{r0, r1, r2, r3}, ids)) return;
  } else {
    it.kvh = x % a.hkv; x /= a.hkv;
    const int gt = x % a.gt; x /= a.gt;
    const int sx = x % a.ss, i = x / a.ss;
    const int lim = visible(a, i, &it.row);
    if (a.prefix && it.kvh == 0 && gt == 0 && sx == 0 && threadIdx.x < 64 && it.row >= 0) {   // what it reads as shared, is it on the same pages?
      const int pr = prefix_row(a, lane), held = ((lim < a.prefix ? lim : a.prefix) + (1 << a.log_ps) - 1) >> a.log_ps;
      bool differ = false;
      for (int j = lane; j < held; j += 64) differ |= pr < 0 || a.table[(size_t)it.row * a.width + j] != a.table[(size_t)pr * a.width + j];
      if (__any(differ) && lane == 0) atomicOr(a.status, (int)ORC_KV_NOT_SHARED);
    }
    const int tiles = (lim - a.prefix + KT - 1) / KT;
    int per = (tiles + a.ss - 1) / a.ss;
    per = (per < 4 ? 4 : per) * KT;   // at least a tile for each wave
    it.k_lo = a.prefix + sx * per;
    it.k_hi = it.k_lo + per < lim ? it.k_lo + per : lim;
    it.part = a.sp + sx;
    it.f0 = i * a.group + gt * 16;
    it.cols = a.group - gt * 16;
    if (it.cols > 16) it.cols = 16;
  }
  keys_items<T, HD, NID>(a, it, room, ids, sm);
}

// One wave per (query, head): lane s holds the weight of part s; then the lanes hold the head's dims, 16 bytes each, and a wave reads 64 * 4 / HD
// parts at a time, the loads of four such groups in flight.
template <typename T, int HD>
__global__ __launch_bounds__(256) void combine_kernel(AttendArgs a) {
  constexpr int LD = HD / 4, G = 64 / LD;     // lanes of a part, parts a wave reads at once
  const int lane = threadIdx.x & 63, sub = lane / LD, d = lane % LD * 4;
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= (long)a.n * a.hq) return;
  const int parts = a.sp + a.ss;
  float m = -INFINITY, l = 0.f;
  if (lane < parts) { m = a.ml[2 * (id * parts + lane)]; l = a.ml[2 * (id * parts + lane) + 1]; }
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* po = a.po + id * parts * HD + d;
  f32x4 v[4];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * G + sub;
      v[u] = *(const f32x4*)(po + (size_t)(s < parts ? s : parts - 1) * HD);
    }
  };
  load(0);
  if (l == 0.f) m = -INFINITY;
  const float mx = wave_max(m);
  const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - mx) * a.c);
  const float sum = wave_sum(l * f);
  for (int s0 = 0; s0 < parts; s0 += 4 * G) {
    if (s0) load(s0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * G + sub;
      const float fs = __shfl(f, s & 63, 64), ls = __shfl(l, s & 63, 64);
      if (s < parts && ls != 0.f) acc += v[u] * fs;   // a part without tokens was not written
    }
  }
#pragma unroll
  for (int o = LD; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], o, 64);
  if (sub) return;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int i = (int)(id / a.hq), head = (int)(id % a.hq);
  u32x2 st = {cvt2<T>(acc[0] * inv, acc[1] * inv), cvt2<T>(acc[2] * inv, acc[3] * inv)};
  if (sum == 0.f && attends(a, i)) st[0] = st[1] = cvt2<T>(NAN, NAN);
  *(u32x2*)((T*)a.o + (size_t)i * a.o_ts + (size_t)head * a.o_hs + d) = st;
}

// how a call is split; the same for the scratch size and the launch
struct Split { bool cols; int mt, gt, sp, ss; };
Split split_of(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  Split s;
  const int group = n_heads / c->n_kv_heads;
  const int64_t cols = (int64_t)n * group;
  // keys_item reads the prefix once for every 16 columns, cols_item for every 128, with fewer and larger workgroups. The second pass of 17 to 32
  // columns is cheap while the first one's pages are in the caches (keys / cols us at 32 columns: 32 K/V heads, 768 shared tokens 18.3 / 20.8, 4k
  // 28.2 / 30.6; 2 heads, 16k 17.4 / 20.9) and is not beyond (32 heads, 8k, 134 MB 42.9 / 43.2; 16k 71.9 / 66.0); more passes cost more (48
  // columns: 8 heads, 4k 15.3 / 15.6, 32k 52.2 / 39.1; 32 heads, 8k 60.3 / 51.1).
  // cols_item reads at most IDS_COLS - 4 pages, of MAX_SP parts at the most.
  const int64_t range = (int64_t)(IDS_COLS - 4) * c->page_size, least_sp = (prefix + range - 1) / range;
  const int64_t bytes = (int64_t)prefix * c->n_kv_heads * c->head_dim * 4;
  s.cols = cols > (bytes > 128 << 20 ? 16 : 32) && least_sp <= MAX_SP;
  const int wide = s.cols ? 128 : 16;
  s.mt = prefix ? (int)((cols + wide - 1) / wide) : 0;
  s.gt = (group + 15) / 16;
  s.sp = 0;
  if (prefix) {
    const int64_t base = (int64_t)c->n_kv_heads * s.mt;
    // cols_item runs two to a CU: 256 items leave every other place to the rows' own tokens, which are bound by memory, not by the matrix cores
    // (us with 256 / 384 / 512 items: 96 rows, 32 heads on 8, 32k shared + 0..2000 own tokens 117 / 127 / 134, + 200 94 / 88 / 95, without own
    // tokens 89 / 82 / 81; 64 rows over 8k + 0..500 31 / 35 / 39; 128 rows, 16 heads on 2, 16k + 0..1000 39 / 44 / 50).
    // keys_item: 512, of 256 keys and more.
    int64_t sp = ((s.cols ? 256 : 512) + base - 1) / base;
    const int64_t most_sp = (prefix + 255) / 256;
    sp = sp < most_sp ? sp : most_sp;
    sp = sp < 1 ? 1 : sp > MAX_SP ? MAX_SP : sp;
    sp = s.cols && sp < least_sp ? least_sp : sp;
    const int unit = s.cols ? UNIT_COLS : UNIT_KEYS;   // as attend_kernel cuts it; no part is empty (201 tiles in 40 parts are 34 of 6)
    const int64_t tiles = (prefix + unit - 1) / unit, per = (tiles + sp - 1) / sp;
    s.sp = (int)((tiles + per - 1) / per);
  }
  const int64_t own = (int64_t)n * c->n_kv_heads * s.gt;
  const int64_t left = (int64_t)c->max_row_pages * c->page_size - prefix;
  int64_t ss = (512 + own - 1) / own;
  const int64_t most_ss = (left + 255) / 256;
  ss = ss < most_ss ? ss : most_ss;
  s.ss = (int)(ss < 1 ? 1 : ss > MAX_SS ? MAX_SS : ss);
  return s;
}

const char* bad_call(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  if (!c) return "null argument";
  if (c->n_kv_heads < 1 || n_heads < 1 || n_heads % c->n_kv_heads) return "n_heads is not a multiple of n_kv_heads";
  if (n < 0 || n > 1024) return "0..1024 queries a call";
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return "page_size is 16, 32, 64 or 128";
  if ((int64_t)c->n_kv_heads * c->page_size * 128 * 2 > 0x7fffffff) return "a page of 2 GiB and more";
  if (c->max_rows < 1 || c->n_pages < 1 || c->max_row_pages < 1 || c->max_row_pages > 1 << 20) return "bad geometry";
  if (prefix < 0 || prefix % c->page_size || (int64_t)prefix > (int64_t)c->max_row_pages * c->page_size)
    return "prefix_tokens is not a multiple of page_size inside a row";
  return nullptr;
}

// 256 threads a workgroup, 32 bits of threads a launch; cols_item counts (query, head, part) in 32 bits
bool too_large(const orc_kv_pages* c, int n, int n_heads, const Split& s) {
  const int64_t items = (int64_t)c->n_kv_heads * s.mt * s.sp + (int64_t)n * c->n_kv_heads * s.gt * s.ss, waves = (int64_t)n * n_heads;
  return items > 0xffffff || (waves + 3) / 4 > 0xffffff || waves * (s.sp + s.ss) > 0x7fffffff;
}
constexpr const char* TOO_LARGE = "too many queries and heads: 2^24 - 1 workgroups and 2^31 - 1 parts at the most";

template <typename T, int HD, bool COLS> hipError_t launch_cols(const AttendArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)(a.hkv * a.mt * a.sp + a.n * a.hkv * a.gt * a.ss);   // (not too_large)
  hipLaunchKernelGGL((attend_kernel<T, HD, COLS>), dim3(grid), dim3(256), 0, s, a);
  if (a.sp + a.ss > 1)
    hipLaunchKernelGGL((combine_kernel<T, HD>), dim3((unsigned)(((int64_t)a.n * a.hq + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename T, int HD> hipError_t launch_hd(const AttendArgs& a, bool cols, hipStream_t s) {
  return cols ? launch_cols<T, HD, true>(a, s) : launch_cols<T, HD, false>(a, s);
}

}  // namespace

extern "C" int64_t orc_kv_attend_ws(const orc_kv_pages* c, int n, int n_heads, int prefix) {
  const char* bad = bad_call(c, n, n_heads, prefix);
  if (bad) return orc_fail("orc_kv_attend_ws", bad);
  const Split s = split_of(c, n < 1 ? 1 : n, n_heads, prefix);
  if (too_large(c, n, n_heads, s)) return orc_fail("orc_kv_attend_ws", TOO_LARGE);
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
  if (too_large(c, n, n_heads, s)) return orc_fail(who, TOO_LARGE);
  if (!q || !out || !rows || !c->kv || !c->table || !c->lens || !c->status || (s.sp + s.ss > 1 && !ws)) return orc_fail(who, "null argument");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)c->kv | (uintptr_t)ws) & 15) return orc_fail(who, "tensors are not aligned to 16 bytes");
  const HeadView vo{out, st[2], st[3], n, n_heads, c->head_dim};
  if (out_meets_q(vo, {q, st[0], st[1], n, n_heads, c->head_dim})) return orc_fail(who, "out lies over q and is not q");
  AttendArgs a;
  const size_t page = (size_t)c->n_kv_heads * c->page_size * c->head_dim;
  const char* kv_end = (const char*)c->kv + (size_t)c->n_layers * 2 * c->n_pages * page * 2;
  if ((const char*)out < kv_end && (const char*)out + ((n - 1) * vo.ts + (n_heads - 1) * vo.hs + c->head_dim) * 2 > (const char*)c->kv)
    return orc_fail(who, "out lies over the pool");
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
  if (c->dtype == 0) e = c->head_dim == 128 ? launch_hd<__bf16, 128>(a, s.cols, hs) : launch_hd<__bf16, 64>(a, s.cols, hs);
  else e = c->head_dim == 128 ? launch_hd<_Float16, 128>(a, s.cols, hs) : launch_hd<_Float16, 64>(a, s.cols, hs);
  return e == hipSuccess ? 0 : orc_fail(who, hipGetErrorString(e));
}
