// Bookkeeping and copies of the paged KV cache (orc_kv_reserve / append / fork / free / compact).
//
// The page table, the rows' lengths and the pages' reference counts live on the device, so a call needs no host round trip and can be captured.
// Everything that has to be decided for a whole call at once (are the lists right, are there enough free pages, which are the lowest)
// is one workgroup of 1024 threads; what moves tokens is a second launch over all CUs that reads the list of copies the first one left.
//
// Such a workgroup is bound by the chain of its loads (lists, lengths, table, counts: about 1 us each, one behind the other) and a dozen barriers, not by
// bytes: reserve 9.7 us for 8 prompts of 6156 tokens, fork 8.4 us for 24 rows of 2 sources, free 4-5 us, compact's two 4.8 us each (medians of 200). Of
// many long rows it is the walk over the table by one CU: fork and free of a row of 2048 pages to 96 rows 320 us. The copies are bound by HBM: append
// 39 us for a layer of those prompts (200 MB, 5.1 TB/s), compact 357 us (1.77 GB, 5.0 TB/s), whole rows of 16-token pages at head dim 64 113 us (547 MB,
// 4.8 TB/s).
#include "../../include/oracle_hip.h"
#include "kernels.h"
#include "mma16.h"

namespace {

constexpr int NT = 1024;
// work[]: 8 header ints, then three lists of n_pages ints and a map of n_pages
enum { W_COUNT = 0, W_LIVE = 1 };

struct Pages {
  char* kv;
  int *table, *lens, *refs, *status, *work;
  int n_layers, n_pages, hkv, ps, log_ps, max_rows, width, head_bytes;   // head_bytes: one token of one head
};

__device__ __forceinline__ int wave_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
// exclusive prefix of v over the workgroup, *total = sum
__device__ int block_scan(int v, int* total, int* sh) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int inc = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  if (w == 0) {
    const int x = lane < NT / 64 ? sh[lane] : 0;
    const int s = wave_scan(x, lane);
    if (lane < NT / 64) sh[lane] = s - x;
    if (lane == NT / 64 - 1) sh[NT / 64] = s;
  }
  __syncthreads();
  *total = sh[NT / 64];
  return sh[w] + inc - v;
}

// The `need` lowest free pages, ascending, to list; false where there are fewer. 16 pages a thread at a time, all their loads in flight at once;
// it stops as soon as it has enough.
__device__ bool lowest_free(const Pages& p, int need, int* list, int* sh) {
  constexpr int PER = 16;
  int found = 0;
  for (int base = 0; base < p.n_pages && found < need; base += NT * PER) {
    const int lo = base + (int)threadIdx.x * PER;
    int r[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) r[j] = p.refs[lo + j < p.n_pages ? lo + j : p.n_pages - 1];
#pragma unroll
    for (int j = 0; j < PER; ++j) mine += lo + j < p.n_pages && r[j] == 0;
    int total, at = found + block_scan(mine, &total, sh);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lo + j < p.n_pages && r[j] == 0) {
        if (at < need) list[at] = lo + j;
        ++at;
      }
    found += total;
  }
  __threadfence_block();
  __syncthreads();
  return found >= need;
}

// the last of n entries whose first[] (ascending) is at most x; entries of no size start where the next does and are passed over
__device__ __forceinline__ int entry_of(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(const Pages& p, int tokens) { return (tokens + p.ps - 1) >> p.log_ps; }

// Entry t of a list of rows, and the tokens of that row (0 where it is outside the table; 0 and 0 behind the list). The loads are asked for before the rows
// are checked: their latency is most of what these kernels take.
__device__ __forceinline__ int row_of(const int* rows, int n) { return (int)threadIdx.x < n ? rows[threadIdx.x] : 0; }
__device__ __forceinline__ int tokens_of(const Pages& p, int r, int n) {
  const int len = p.lens[r >= 0 && r < p.max_rows ? r : 0];
  return (int)threadIdx.x < n && r >= 0 && r < p.max_rows ? len : 0;
}
// Whether the threads' rows are rows of the table, each once. seen: a bit per row (max_rows <= 65536), cleared here.
__device__ int check_rows(const Pages& p, int r, int n, unsigned* seen) {
  for (int i = threadIdx.x; i < (p.max_rows + 31) / 32; i += NT) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  if ((int)threadIdx.x < n) {
    if (r < 0 || r >= p.max_rows) bad = ORC_KV_BAD_ROW;
    else if (atomicOr(&seen[r >> 5], 1u << (r & 31)) >> (r & 31) & 1) bad = ORC_KV_ROW_TWICE;
  }
  return bad;
}

// all threads' bits together
__device__ int block_or(int v, int* sh) {
  if (!__syncthreads_or(v)) return 0;
  if (threadIdx.x == 0) sh[0] = 0;
  __syncthreads();
  if (v) atomicOr(&sh[0], v);
  __syncthreads();
  const int r = sh[0];
  __syncthreads();
  return r;
}

__global__ __launch_bounds__(NT) void reserve_kernel(Pages p, const int* rows, const int* counts, int n, int* slots, int total) {
  __shared__ int sh[NT / 64 + 1];
  __shared__ unsigned seen[2048];
  __shared__ int tok0[NT], page0[NT], from[NT], of[NT];   // of every list entry: first new token, first new page, tokens held before, row
  const int t = threadIdx.x;
  const int r = row_of(rows, n), more = counts ? row_of(counts, n) : 1, old = tokens_of(p, r, n);
  int bad = check_rows(p, r, n, seen), add = 0;
  if (t < n && !bad) {
    add = more;
    if (add < 0 || add > total) bad = ORC_KV_BAD_COUNT;   // (more than `total` fails below anyway; here it bounds the sums)
    else if (old < 0 || (long)old + add > (long)p.width * p.ps) bad = ORC_KV_ROW_FULL;
    if (bad) add = 0;
  }
  int part = 0;   // the page that the row's next token goes to, where it has been begun: looked at behind the sums, its load meanwhile in flight
  if (add > 0 && (old & (p.ps - 1))) part = p.table[(size_t)r * p.width + (old >> p.log_ps)];
  bad = block_or(bad, sh);
  int need_all = 0, add_all = 0, at = 0, first = 0;
  if (!bad) {
    first = block_scan(add, &add_all, sh);
    if (add_all > total) bad = ORC_KV_BAD_COUNT;
  }
  int* list = p.work + 8;
  if (!bad) {
    // fewer than 2^20 pages (2^20 tokens in pages of 16, one more a row): what is above counts the bad ones, without a barrier more
    at = block_scan(pages_of(p, old + add) - pages_of(p, old) + (part < 0 || part >= p.n_pages ? 1 << 20 : 0), &need_all, sh);
    if (need_all >> 20) bad = ORC_KV_BAD_PAGE;
    else if (need_all > p.n_pages || !lowest_free(p, need_all, list, sh)) bad = ORC_KV_POOL_FULL;
  }
  if (bad) {   // the same for all threads
    if (t == 0) atomicOr(p.status, bad);
    for (int i = t; i < total; i += NT) slots[i] = -1;
    return;
  }
  tok0[t] = first; page0[t] = at; from[t] = old; of[t] = r;
  __syncthreads();
  for (int x = t; x < need_all; x += NT) {
    const int e = entry_of(page0, n, x), page = list[x];
    p.refs[page] = 1;
    p.table[(size_t)of[e] * p.width + pages_of(p, from[e]) + x - page0[e]] = page;
  }
  if (t < n) p.lens[r] = old + add;
  for (int i = t; i < total; i += NT) {
    int s = -1;
    if (i < add_all) {
      const int e = entry_of(tok0, n, i), pos = from[e] + i - tok0[e], j = (pos >> p.log_ps) - pages_of(p, from[e]);   // j < 0: the part page
      const int page = j < 0 ? p.table[(size_t)of[e] * p.width + (pos >> p.log_ps)] : list[page0[e] + j];
      s = page * p.ps + (pos & (p.ps - 1));
    }
    slots[i] = s;
  }
}

// 16-byte pieces of one token (all heads, K then V) over a workgroup's threads
__global__ __launch_bounds__(256) void append_kernel(Pages p, const int* slots, int total, const char* k, const char* v, long k_ts, long k_hs,
                                                     long v_ts, long v_hs, char* kd, char* vd) {
  const int per_head = p.head_bytes >> 4, per = p.hkv * per_head;
  const long all = (long)total * per * 2;
  for (long x = (long)blockIdx.x * 256 + threadIdx.x; x < all; x += (long)gridDim.x * 256) {
    const int tok = (int)(x / (2 * per)), y = (int)(x % (2 * per)), z = y < per ? y : y - per;
    const int head = z / per_head, piece = z % per_head;
    const int s = slots[tok];
    if (s < 0 || (s >> p.log_ps) >= p.n_pages) continue;
    const size_t dst = (((size_t)(s >> p.log_ps) * p.hkv + head) * p.ps + (s & (p.ps - 1))) * p.head_bytes + piece * 16;
    const u32x4 val = y < per ? *(const u32x4*)(k + tok * k_ts + head * k_hs + piece * 16) : *(const u32x4*)(v + tok * v_ts + head * v_hs + piece * 16);
    *(u32x4*)((y < per ? kd : vd) + dst) = val;
  }
}

__global__ __launch_bounds__(NT) void fork_kernel(Pages p, const int* src, const int* dst, int n, int n_tokens, int share) {
  __shared__ int sh[NT / 64 + 1];
  __shared__ unsigned seen[2048];
  __shared__ int src_of[NT], dst_of[NT], len_of[NT], page0[NT], most_sh;   // of every pair; page0: its first fresh page
  const int t = threadIdx.x;
  if (t == 0) most_sh = 0;
  const int d = row_of(dst, n), s = row_of(src, n), held = tokens_of(p, d, n), source = tokens_of(p, s, n);
  int bad = check_rows(p, d, n, seen), len = 0;
  __syncthreads();
  if (t < n && !bad) {
    if (s < 0 || s >= p.max_rows) bad = ORC_KV_BAD_ROW;
    else if (seen[s >> 5] >> (s & 31) & 1) bad = ORC_KV_ROW_TWICE;   // a source that is also a destination
    else if (held != 0) bad = ORC_KV_NOT_EMPTY;
    else {
      len = source;
      if (n_tokens >= 0 && n_tokens < len) len = n_tokens;
      if (len < 0 || len > p.width * p.ps) { bad = ORC_KV_BAD_COUNT; len = 0; }
    }
  }
  const int used = pages_of(p, len), keep = share ? len >> p.log_ps : 0;
  if (used) atomicMax(&most_sh, used);   // (1024 threads on one LDS word would take 2 us)
  bad = block_or(bad, sh);
  int need_all = 0, at = 0;
  if (!bad) at = block_scan(used - keep, &need_all, sh);
  src_of[t] = s; dst_of[t] = d; len_of[t] = len; page0[t] = at;
  __syncthreads();
  const int most = most_sh;   // the pairs' pages as a grid of n x most
  if (!bad) {
    int off = 0;
    for (int x = t; x < n * most; x += NT) {
      const int i = x / most, j = x - i * most;
      if (j >= pages_of(p, len_of[i])) continue;
      const int page = p.table[(size_t)src_of[i] * p.width + j];
      if (page < 0 || page >= p.n_pages) off = ORC_KV_BAD_PAGE;
    }
    bad = block_or(off, sh);
  }
  // the copies: to work[8 + c], from work[8 + n_pages + c], tokens work[8 + 2 n_pages + c]
  int* list = p.work + 8;
  if (!bad && (need_all > p.n_pages || !lowest_free(p, need_all, list, sh))) bad = ORC_KV_POOL_FULL;
  if (bad) {
    if (t == 0) { atomicOr(p.status, bad); p.work[W_COUNT] = 0; }
    return;
  }
  for (int x = t; x < n * most; x += NT) {
    const int i = x / most, j = x - i * most, tokens = len_of[i];
    if (j >= pages_of(p, tokens)) continue;
    const int from = p.table[(size_t)src_of[i] * p.width + j], kept = share ? tokens >> p.log_ps : 0;
    int to = from;
    if (j < kept) {
      atomicAdd(&p.refs[from], 1);
    } else {
      const int c = page0[i] + j - kept;
      to = list[c];
      p.refs[to] = 1;
      list[p.n_pages + c] = from;
      list[2 * p.n_pages + c] = tokens - j * p.ps < p.ps ? tokens - j * p.ps : p.ps;
    }
    p.table[(size_t)dst_of[i] * p.width + j] = to;
  }
  if (t < n) p.lens[d] = len;
  if (t == 0) p.work[W_COUNT] = need_all;
}

// The listed copies, work[W_COUNT] of them, for every layer's K and V: tokens from a page of `from` to a page of `to`. A unit is one page of
// one plane; tokens behind the last are left as they were.
__global__ __launch_bounds__(256) void copy_kernel(const char* from, char* to, const int* work, int list, int planes, int n_from, int n_to,
                                                   int hkv, int ps, int head_bytes) {
  const int count = work[W_COUNT];
  const size_t page = (size_t)hkv * ps * head_bytes;
  for (long u = blockIdx.x; u < (long)count * planes; u += gridDim.x) {
    const int c = (int)(u / planes), plane = (int)(u % planes);
    const int d = work[8 + c], s = work[8 + list + c], tokens = work[8 + 2 * list + c];
    const char* sp = from + ((size_t)plane * n_from + s) * page;
    char* dp = to + ((size_t)plane * n_to + d) * page;
    const int seg = tokens * head_bytes >> 4, heads = tokens == ps ? 1 : hkv;
    const int len = tokens == ps ? (int)(page >> 4) : seg;
    for (int hd = 0; hd < heads; ++hd) {
      const size_t off = (size_t)hd * ps * head_bytes;
      for (int x = threadIdx.x; x < len; x += 256) ((u32x4*)(dp + off))[x] = ((const u32x4*)(sp + off))[x];
    }
  }
}

__global__ __launch_bounds__(NT) void free_kernel(Pages p, const int* rows, int n) {
  __shared__ int sh[NT / 64 + 1];
  __shared__ unsigned seen[2048];
  __shared__ int pages[NT], of[NT], most_sh;   // of every row: its pages, its place in the table
  const int t = threadIdx.x;
  if (t == 0) most_sh = 0;
  const int r = row_of(rows, n), len = tokens_of(p, r, n);
  int bad = check_rows(p, r, n, seen);
  bad = block_or(bad, sh);
  if (bad) {
    if (t == 0) atomicOr(p.status, bad);
    return;
  }
  // Up to the longest row, not the table's width (64 rows of 13 pages in a table 4096 wide: 108 -> 7 us; of 2000: 186 -> 39; 16 of 13 in 16: 6.2 -> 6.6).
  const int used = len <= 0 ? 0 : len < p.width * p.ps ? pages_of(p, len) : p.width;
  if (used) atomicMax(&most_sh, used);
  pages[t] = used;
  of[t] = r;
  __syncthreads();
  const int most = most_sh;
  for (int x = t; x < n * most; x += NT) {
    const int i = x / most, j = x - i * most;
    if (j >= pages[i]) continue;
    int* e = &p.table[(size_t)of[i] * p.width + j];
    const int page = *e;
    if (page >= 0 && page < p.n_pages) atomicSub(&p.refs[page], 1);
    *e = -1;
  }
  if (t < n) p.lens[r] = 0;
}

// where every held page goes: map[page] (work list 3) and the copies; in place only pages behind the last to keep move
__global__ __launch_bounds__(NT) void compact_plan_kernel(Pages p, int n_to, int* to_status, int in_place) {
  __shared__ int sh[NT / 64 + 1];
  const int per = (p.n_pages + NT - 1) / NT, lo = threadIdx.x * per;
  const int hi = lo + per < p.n_pages ? lo + per : p.n_pages;
  int* map = p.work + 8 + 3 * p.n_pages;
  int mine = 0;
  for (int i = lo; i < hi; ++i) mine += p.refs[i] > 0;
  int live, at = block_scan(mine, &live, sh);
  if (live > n_to) {
    if (threadIdx.x == 0) { atomicOr(to_status, (int)ORC_KV_POOL_FULL); p.work[W_COUNT] = 0; p.work[W_LIVE] = -1; }
    return;
  }
  if (!in_place) {
    for (int i = lo; i < hi; ++i) {
      const bool held = p.refs[i] > 0;
      map[i] = held ? at : -1;
      if (held) {
        p.work[8 + at] = at;
        p.work[8 + p.n_pages + at] = i;
        p.work[8 + 2 * p.n_pages + at] = p.ps;
        ++at;
      }
    }
    if (threadIdx.x == 0) { p.work[W_COUNT] = live; p.work[W_LIVE] = live; }
    return;
  }
  int movers = 0, holes = 0;
  for (int i = lo; i < hi; ++i) {
    movers += p.refs[i] > 0 && i >= live;
    holes += p.refs[i] <= 0 && i < live;
  }
  int n_move, n_hole;
  int am = block_scan(movers, &n_move, sh), ah = block_scan(holes, &n_hole, sh);
  for (int i = lo; i < hi; ++i) {
    const bool held = p.refs[i] > 0;
    map[i] = held ? i : -1;
    if (held && i >= live) { p.work[8 + p.n_pages + am] = i; p.work[8 + 2 * p.n_pages + am] = p.ps; ++am; }
    if (!held && i < live) p.work[8 + ah++] = i;
  }
  __threadfence_block();
  __syncthreads();
  for (int c = threadIdx.x; c < n_move; c += NT) {
    const int s = p.work[8 + p.n_pages + c], d = p.work[8 + c];
    map[s] = d;
    p.refs[d] = p.refs[s];
    p.refs[s] = 0;
  }
  if (threadIdx.x == 0) { p.work[W_COUNT] = n_move; p.work[W_LIVE] = live; }
}

// the rows of `to` (the same cache, or the other one) by the map
__global__ __launch_bounds__(256) void compact_table_kernel(Pages p, Pages to, int in_place) {
  if (p.work[W_LIVE] < 0) return;
  const int* map = p.work + 8 + 3 * p.n_pages;
  const long step = (long)gridDim.x * 256, x0 = (long)blockIdx.x * 256 + threadIdx.x;
  for (long x = x0; x < (long)p.max_rows * p.width; x += step) {
    const int page = p.table[x];
    to.table[x] = page >= 0 && page < p.n_pages ? map[page] : -1;
  }
  if (in_place) return;
  for (long x = x0; x < p.max_rows; x += step) to.lens[x] = p.lens[x];
  const int live = p.work[W_LIVE];
  for (long x = x0; x < to.n_pages; x += step) to.refs[x] = x < live ? p.refs[p.work[8 + p.n_pages + x]] : 0;
}

const char* bad_cache(const orc_kv_pages* c) {
  if (!c || !c->kv || !c->table || !c->lens || !c->refs || !c->status || !c->work) return "null argument";
  if (c->n_layers < 1 || c->n_pages < 1 || c->n_kv_heads < 1 || c->max_row_pages < 1) return "bad geometry";
  if (c->max_rows < 1 || c->max_rows > 65536) return "1..65536 rows a cache";
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return "page_size is 16, 32, 64 or 128";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim is 64 or 128";
  if (c->dtype != 0 && c->dtype != 1) return "dtype is 0 (bf16) or 1 (fp16)";
  if ((int64_t)c->n_kv_heads * c->page_size * c->head_dim * 2 > 0x7fffffff) return "a page of 2 GiB and more";
  if ((int64_t)c->n_pages * c->page_size > 0x7fffffff) return "more than 2^31 - 1 tokens in the pool";
  if (c->max_row_pages > 1 << 20) return "more than 2^20 pages a row";   // 1024 rows' pages add up in 32 bits
  if ((uintptr_t)c->kv & 15) return "kv is not aligned to 16 bytes";
  return nullptr;
}
Pages dev(const orc_kv_pages* c) {
  Pages p;
  p.kv = (char*)c->kv; p.table = c->table; p.lens = c->lens; p.refs = c->refs; p.status = c->status; p.work = c->work;
  p.n_layers = c->n_layers; p.n_pages = c->n_pages; p.hkv = c->n_kv_heads; p.ps = c->page_size; p.log_ps = __builtin_ctz(c->page_size);
  p.max_rows = c->max_rows; p.width = c->max_row_pages; p.head_bytes = c->head_dim * 2;
  return p;
}
bool overlap(const void* x, int64_t nx, const void* y, int64_t ny) { return (const char*)x < (const char*)y + ny && (const char*)y < (const char*)x + nx; }
int done(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : orc_fail(who, hipGetErrorString(e));
}

}  // namespace

extern "C" int orc_kv_reserve(const orc_kv_pages* c, const int32_t* rows, const int32_t* counts, int n, int32_t* slots, int total, void* stream) {
  const char* who = "orc_kv_reserve";
  if (const char* bad = bad_cache(c)) return orc_fail(who, bad);
  if (n < 0 || n > NT) return orc_fail(who, "0..1024 rows a call");
  if (total < 0 || total > 1 << 20) return orc_fail(who, "0..2^20 tokens a call");   // 1024 counts add up in 32 bits
  if (n == 0 && total == 0) return 0;
  if ((n > 0 && !rows) || (total > 0 && !slots)) return orc_fail(who, "null argument");
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(NT), 0, (hipStream_t)stream, dev(c), rows, counts, n, slots, total);
  return done(who);
}

extern "C" int orc_kv_append(const orc_kv_pages* c, int layer, const int32_t* slots, int total, const void* k, const void* v, const int64_t* st,
                             void* stream) {
  const char* who = "orc_kv_append";
  if (const char* bad = bad_cache(c)) return orc_fail(who, bad);
  if (layer < 0 || layer >= c->n_layers) return orc_fail(who, "layer outside the cache");
  if (total < 0 || !st) return orc_fail(who, "bad argument");
  for (int i = 0; i < 4; ++i)
    if (st[i] < 0 || st[i] % 8) return orc_fail(who, "strides are not multiples of 8 elements");
  if (total == 0) return 0;
  if (!slots || !k || !v) return orc_fail(who, "null argument");
  if (((uintptr_t)k | (uintptr_t)v) & 15) return orc_fail(who, "tensors are not aligned to 16 bytes");
  const Pages p = dev(c);
  const size_t plane = (size_t)p.n_pages * p.hkv * p.ps * p.head_bytes;
  char* kd = p.kv + (size_t)layer * 2 * plane;
  const int64_t pieces = (int64_t)total * p.hkv * (p.head_bytes >> 4) * 2;
  const int64_t grid = (pieces + 255) / 256;
  hipLaunchKernelGGL(append_kernel, dim3((unsigned)(grid < 8192 ? grid : 8192)), dim3(256), 0, (hipStream_t)stream, p, slots, total, (const char*)k,
                     (const char*)v, st[0] * 2, st[1] * 2, st[2] * 2, st[3] * 2, kd, kd + plane);
  return done(who);
}

extern "C" int orc_kv_fork(const orc_kv_pages* c, const int32_t* src, const int32_t* dst, int n, int n_tokens, int share, void* stream) {
  const char* who = "orc_kv_fork";
  if (const char* bad = bad_cache(c)) return orc_fail(who, bad);
  if (n < 0 || n > NT) return orc_fail(who, "0..1024 rows a call");
  if (n == 0) return 0;
  if (!src || !dst) return orc_fail(who, "null argument");
  const Pages p = dev(c);
  hipLaunchKernelGGL(fork_kernel, dim3(1), dim3(NT), 0, (hipStream_t)stream, p, src, dst, n, n_tokens, share);
  hipLaunchKernelGGL(copy_kernel, dim3(2048), dim3(256), 0, (hipStream_t)stream, p.kv, p.kv, p.work, p.n_pages, p.n_layers * 2, p.n_pages,
                     p.n_pages, p.hkv, p.ps, p.head_bytes);
  return done(who);
}

extern "C" int orc_kv_free(const orc_kv_pages* c, const int32_t* rows, int n, void* stream) {
  const char* who = "orc_kv_free";
  if (const char* bad = bad_cache(c)) return orc_fail(who, bad);
  if (n < 0 || n > NT) return orc_fail(who, "0..1024 rows a call");
  if (n == 0) return 0;
  if (!rows) return orc_fail(who, "null argument");
  hipLaunchKernelGGL(free_kernel, dim3(1), dim3(NT), 0, (hipStream_t)stream, dev(c), rows, n);
  return done(who);
}

extern "C" int orc_kv_compact(const orc_kv_pages* c, const orc_kv_pages* into, void* stream) {
  const char* who = "orc_kv_compact";
  if (const char* bad = bad_cache(c)) return orc_fail(who, bad);
  const bool in_place = !into;
  if (!in_place) {
    if (const char* bad = bad_cache(into)) return orc_fail(who, bad);
    if (into->n_layers != c->n_layers || into->n_kv_heads != c->n_kv_heads || into->page_size != c->page_size || into->head_dim != c->head_dim ||
        into->dtype != c->dtype || into->max_rows != c->max_rows || into->max_row_pages != c->max_row_pages)
      return orc_fail(who, "the caches differ in more than n_pages");
    const int64_t page = (int64_t)c->n_layers * 2 * c->n_kv_heads * c->page_size * c->head_dim * 2;
    if (overlap(into->kv, into->n_pages * page, c->kv, c->n_pages * page) || overlap(into->refs, into->n_pages * 4ll, c->refs, c->n_pages * 4ll) ||
        overlap(into->table, c->max_rows * 4ll * c->max_row_pages, c->table, c->max_rows * 4ll * c->max_row_pages) ||
        overlap(into->lens, c->max_rows * 4ll, c->lens, c->max_rows * 4ll))
      return orc_fail(who, "the caches share memory");
  }
  const Pages p = dev(c), q = in_place ? p : dev(into);
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(NT), 0, s, p, q.n_pages, q.status, in_place ? 1 : 0);
  const int64_t entries = (int64_t)p.max_rows * p.width, grid = (entries + 255) / 256;
  hipLaunchKernelGGL(compact_table_kernel, dim3((unsigned)(grid < 1024 ? grid : 1024)), dim3(256), 0, s, p, q, in_place ? 1 : 0);
  hipLaunchKernelGGL(copy_kernel, dim3(2048), dim3(256), 0, s, p.kv, q.kv, p.work, p.n_pages, p.n_layers * 2, p.n_pages, q.n_pages, p.hkv, p.ps,
                     p.head_bytes);
  return done(who);
}
