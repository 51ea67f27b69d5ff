// One wave's part of attention over 64-key tiles in LDS: 32 query columns, running maximum, sum and output in registers. Used by the kernels of
// attn_packed.hip (prompts) and attn_paged.hip (a prefix that many queries share).
//
// Orientation (no value crosses lanes between the two products):
//   S^T = K . Q^T    A = 32 keys x 16 from LDS, B = the wave's 32 query columns held in registers
//                    -> lane (q = lane & 31, h = lane >> 5) holds keys 8 (i / 4) + 4 h + i % 4 of its query, i = 0..15
//   O^T = V^T . P^T  the k-slots (h, j) of the product are DEFINED as the keys the lane holds: P is its own registers rounded to 16 bits,
//                    V^T comes by the transposing LDS read in that order.
// p = exp2(c (s - m)) with c = scale * log2(e). m is raised (and o, l rescaled, a wave-uniform branch) only where a tile's maximum exceeds it by
// more than 8 / c: p then stays below 2^8, whose rounding to 16 bits is as exact relatively as below 1, and the 64 multiplies of a
// rescale are spent on few tiles. (bf16 outputs against 64 bits, root mean square: 0.0019 raised at every tile, 0.0022 so.) p is rounded to 16 bits, half
// a step, because the product with V takes 16-bit operands; its sum l is not.
//
// Bound by the SIMDs' issue: a 64-key tile is 32 products of 32 cycles at head dim 128 (16 at 64) and some 280 (190) vector instructions,
// 32 of them exponentials, which share the wave's issue slots with the products. What it reaches is with the kernels.
#pragma once
#include <type_traits>

#include "mma16.h"

// A tile image: 64 rows (keys) of HD values, 16-byte chunk ch of a row at place swz(key, ch), an involution. The 8 lanes of a ds_read_b128 phase
// (8 keys, one chunk) and the 4 keys x 64 bytes of half a transposing read then fall on different banks. LDS-DMA writes lane-linearly, so the
// permutation is applied to the lanes' source addresses.
template <int HD> struct Tile64 {
  static constexpr int KEYS = 64, ROWB = HD * 2, CH = HD / 8, BYTES = KEYS * ROWB;
  static __device__ __forceinline__ int swz_k(int key, int ch) { return HD == 128 ? ch ^ (key & 15) : ch ^ ((key >> 1) & 7); }
  static __device__ __forceinline__ int swz_v(int key, int ch) { return HD == 128 ? ch ^ ((key & 3) << 2) : ch ^ (((key >> 1) & 1) << 2); }
};

template <typename T, int HD> struct Flash32 {
  typedef typename Mma<T>::v8 v8;
  typedef Tile64<HD> Tile;
  v8 qf[HD / 16];
  f32x16 o[HD / 32];
  float m, l;             // l: over the lane's own keys, the other half's are added in total()
  int ka[HD / 16], va[HD / 32];   // byte places of the lane's K chunk (keys 0..31) and V piece (keys 0..15) in the tile images

  __device__ __forceinline__ void init(const T* q, int lane) {   // q: the lane's query row
    const int c32 = lane & 31, h = lane >> 5, vr = 4 * h + ((lane & 15) >> 2);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      qf[kk] = *(const v8*)(q + h * 8 + kk * 16);
      ka[kk] = c32 * Tile::ROWB + (Tile::swz_k(c32, kk * 2 + h) << 4);
    }
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
      va[dt] = vr * Tile::ROWB + (Tile::swz_v(vr, dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) << 4) + (lane & 1) * 8;
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) o[dt] = zero();
    m = -INFINITY;
    l = 0.f;
  }
  // scores of keys 32 b .. 32 b + 31 of a tile
  __device__ __forceinline__ f32x16 scores(const char* sK, int b) const {
    f32x16 s = zero();
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) s = score(sK, b, kk, s);
    return s;
  }
  static __device__ __forceinline__ f32x16 zero() {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    return s;
  }
  __device__ __forceinline__ f32x16 score(const char* sK, int b, int kk, f32x16 s) const {
    return Mma<T>::m32(*(const v8*)(sK + ka[kk] + b * 32 * Tile::ROWB), qf[kk], s);
  }
  // key of s[b][i] inside the tile
  static __device__ __forceinline__ int key_of(int b, int i, int h) { return b * 32 + 8 * (i >> 2) + 4 * h + (i & 3); }

  __device__ __forceinline__ float largest(const f32x16 (&s)[2]) const {
    float tm = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) tm = fmaxf(tm, s[b][i]);
    return fmaxf(tm, __shfl_xor(tm, 32, 64));
  }
  __device__ __forceinline__ void raise(float tm, float c) {   // tm: the tile's maximum
    if (__any((tm - m) * c > 8.f)) {   // -inf - -inf: a column that has seen no key yet, and sees none here
      const float m_new = fmaxf(m, tm), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) o[dt] *= alpha;
    }
  }
  __device__ __forceinline__ float base(float c) const { return m == -INFINITY ? 0.f : -m * c; }
  // p of 32 keys, mc = base(c); pf: [16-key group][two keys a register]
  __device__ __forceinline__ void weights(const f32x16& s, float c, float mc, u32x4* pf) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i], c, mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[i + 1], c, mc));
      l += p0 + p1;
      pf[i >> 3][(i & 7) >> 1] = cvt2<T>(p0, p1);
    }
  }
  __device__ __forceinline__ void values(const char* sV, const u32x4 (&pf)[4]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v8 p8 = __builtin_bit_cast(v8, pf[g]);
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) {
        const char* p = sV + va[dt] + g * 16 * Tile::ROWB;
        o[dt] = Mma<T>::m32(join8<T>(lds_tr16<T>(p), lds_tr16<T>(p + 8 * Tile::ROWB)), p8, o[dt]);
      }
    }
  }
  // values() for a tile that may hold infinities or NaN where a query does not look: there 0 times the value would not be 0. Such values are left out of
  // the product, and each one that a query sees (keys up to `sees` of the tile) marks its dim by what it adds: +inf, -inf, or both for NaN.
  __device__ __forceinline__ void values_careful(const char* sV, const u32x4 (&pf)[4], int sees, int h) {
    constexpr unsigned INF = Mma<T>::BF16 ? 0x7f80u : 0x7c00u, ONE = Mma<T>::BF16 ? 0x3f80u : 0x3c00u;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
      f32x16 up = zero(), down = zero();
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const char* p = sV + va[dt] + g * 16 * Tile::ROWB;
        const u32x2 a = lds_tr16<T>(p), b = lds_tr16<T>(p + 8 * Tile::ROWB);
        const u32x4 raw = {a[0], a[1], b[0], b[1]};
        u32x4 clean, pu, pd, see;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          clean[j] = pu[j] = pd[j] = see[j] = 0;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const unsigned u = raw[j] >> (16 * x) & 0xffffu;
            const bool odd = (u & INF) == INF, nan = odd && (u & 0x7fffu) != INF;
            clean[j] |= (odd ? 0u : u) << (16 * x);
            pu[j] |= (odd && (nan || !(u & 0x8000u)) ? ONE : 0u) << (16 * x);
            pd[j] |= (odd && (nan || (u & 0x8000u)) ? ONE : 0u) << (16 * x);
            see[j] |= (key_of(g >> 1, (g & 1) * 8 + 2 * j + x, h) <= sees ? ONE : 0u) << (16 * x);
          }
        }
        o[dt] = Mma<T>::m32(__builtin_bit_cast(v8, clean), __builtin_bit_cast(v8, pf[g]), o[dt]);
        up = Mma<T>::m32(__builtin_bit_cast(v8, pu), __builtin_bit_cast(v8, see), up);
        down = Mma<T>::m32(__builtin_bit_cast(v8, pd), __builtin_bit_cast(v8, see), down);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (up[i] > 0.f) o[dt][i] += INFINITY;
        if (down[i] > 0.f) o[dt][i] -= INFINITY;
      }
    }
  }
  __device__ __forceinline__ bool finite() const {
    float z = 0.f;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) z = fmaf(o[dt][i], 0.f, z);
    return z == 0.f;
  }
  // adds the tile: scores s (masked ones -inf), values at sV
  __device__ __forceinline__ void add(const char* sV, const f32x16 (&s)[2], float c) {
    raise(largest(s), c);
    u32x4 pf[4];
    const float mc = base(c);
    weights(s[0], c, mc, pf);
    weights(s[1], c, mc, pf + 2);
    values(sV, pf);
  }
  __device__ __forceinline__ float total() const { return l + __shfl_xor(l, 32, 64); }

  // The wave's 32 rows out of the registers, by way of LDS (room: 32 rows, nobody else's): a lane holds 4 values here and there of its row, and stored
  // from there an instruction would touch 32 rows with 8 or 16 bytes each. store(row, byte, 16 bytes) is called for whole rows, the lanes of
  // an instruction side by side. F32: the sums as they are; else times `inv`, rounded.
  template <bool F32, typename Store> __device__ __forceinline__ void rows(char* room, int lane, float inv, Store store) const {
    constexpr int RB = HD * (F32 ? 4 : 2), CHR = RB / 16, MASK = CHR < 16 ? CHR - 1 : 15;
    const int q = lane & 31, h = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        if constexpr (F32) {
          const int ch = dt * 8 + i / 2 + h;
          *(f32x4*)(room + q * RB + ((ch ^ (q & MASK)) << 4)) = f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
        } else {
          const int ch = dt * 4 + i / 4;
          *(u32x2*)(room + q * RB + ((ch ^ (q & MASK)) << 4) + h * 8) =
              u32x2{cvt2<T>(o[dt][i] * inv, o[dt][i + 1] * inv), cvt2<T>(o[dt][i + 2] * inv, o[dt][i + 3] * inv)};
        }
      }
#pragma unroll
    for (int x = 0; x < 32 * CHR / 64; ++x) {
      const int row = x * (64 / CHR) + lane / CHR, ch = lane % CHR;
      store(row, ch * 16, *(const u32x4*)(room + row * RB + ((ch ^ (row & MASK)) << 4)));
    }
  }
};

// The LDS images of even and odd tiles. Four arrays of their own, not one: the compiler then sees that a transposing read of one does not touch what the
// DMA in flight writes, and does not wait for that DMA in front of it.
struct Images {
  char *k0, *k1, *v0, *v1;
  __device__ __forceinline__ char* of(int w) const { return w == 0 ? k0 : w == 1 ? k1 : w == 2 ? v0 : v1; }   // behind the loop: a wave's own
};

// The loop over the tiles of a workgroup of 4 waves, keys asked for two tiles ahead and values one. Iteration t waits for its values and the next
// tile's keys, then a barrier (the waves are through with tile t - 1). The products of tile t + 1's scores stand between the exponentials of
// tile t, so the matrix cores work through the softmax, and the DMA instructions stand between the products: issued in one go they held the
// wave up for 1300 of 3700 cycles an iteration (the path to L1 takes 64 bytes a cycle, a tile is 32 KiB).
// All waves make all `tiles` iterations, a wave computes in the first `mine` of them. src supplies
//   RND                  DMA instructions a wave issues for an image
//   K(t, r, to), V(...)  the r-th of them for a tile; t >= tiles: any tile, it is not read
//   mask_last(t, s)      sets the scores of keys that are not to be seen to -inf in the wave's last tile; in the others all are seen
// (A mask or a test inside the steps would cost registers the pipeline does not have: 256 are in use at head dim 128.)
template <typename T, int HD, typename Src>
__device__ __forceinline__ void flash_loop(Flash32<T, HD>& f, Src& src, const Images& im, int tiles, int mine, float c) {
  typedef std::integral_constant<int, 0> even;
  typedef std::integral_constant<int, 1> odd;
  constexpr int RND = Src::RND, NK = HD / 16, EVERY = NK / RND;
  auto arrive = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  auto fetch = [&](int t, auto par) {   // what iteration t asks for
    constexpr int PAR = decltype(par)::value;
#pragma unroll
    for (int r = 0; r < RND; ++r) src.K(t + 2, r, PAR ? im.k1 : im.k0);
#pragma unroll
    for (int r = 0; r < RND; ++r) src.V(t + 1, r, PAR ? im.v0 : im.v1);
  };
  float tm = 0.f;
  // tile t, whose scores are in s; the next tile's go to n
  auto step = [&](int t, const f32x16 (&s)[2], f32x16 (&n)[2], auto par) {
    constexpr int PAR = decltype(par)::value;
    arrive();
    f.raise(tm, c);
    const float mc = f.base(c);
    const char* sK = PAR ? im.k0 : im.k1;
    u32x4 pf[4];
    src.next(t);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      n[b] = f.zero();
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        n[b] = f.score(sK, b, kk, n[b]);
        if (kk % EVERY == EVERY - 1) {
          if (b == 0) src.K(t + 2, kk / EVERY, PAR ? im.k1 : im.k0);
          else src.V(t + 1, kk / EVERY, PAR ? im.v0 : im.v1);
        }
      }
      f.weights(s[b], c, mc, pf + 2 * b);
    }
    f.values(PAR ? im.v1 : im.v0, pf);
    tm = f.largest(n);
  };
  auto finish = [&](int t, f32x16 (&s)[2], auto par) {
    constexpr int PAR = decltype(par)::value;
    arrive();
    if (t + 1 < tiles) {
      src.next(t);
      fetch(t, par);
    }
    src.mask_last(t, s);
    f.add(PAR ? im.v1 : im.v0, s, c);
  };
  src.next(-2);
#pragma unroll
  for (int r = 0; r < RND; ++r) src.K(0, r, im.k0);
  src.next(-1);
#pragma unroll
  for (int r = 0; r < RND; ++r) src.V(0, r, im.v0);
#pragma unroll
  for (int r = 0; r < RND; ++r) src.K(1, r, im.k1);
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * RND) : "memory");   // the first keys (and queries): the scores need no more
  __syncthreads();
  int t = 0;
  if (mine > 0) {
    f32x16 s[2] = {f.scores(im.k0, 0), f.scores(im.k0, 1)}, n[2];
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
    arrive();
    if (t + 1 == tiles) break;
    src.next(t);
    if (t & 1) fetch(t, odd());
    else fetch(t, even());
  }
  arrive();   // what was asked for behind the last tile
}
