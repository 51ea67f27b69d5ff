// C ABI (include/oracle_hip.h) + stage orchestration: weights resident in packed form, KV cache and
// workspace pre-allocated, every stage a short sequence of the kernels in gemm/gemv/attn/norm/misc.hip.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <map>
#include <string>
#include <vector>

#include "../../include/oracle_hip.h"
#include "common.h"
#include "kernels.h"

static thread_local char g_err[512] = "";
extern "C" const char* orc_last_error(void) { return g_err; }
extern "C" int orc_abi_version(void) { return 1; }

int orc_fail(const char* what, const char* detail) {
  snprintf(g_err, sizeof(g_err), "%s: %s", what, detail);
  return -1;
}
static int fail(const char* what, const char* detail) { return orc_fail(what, detail); }
#define HIPCHK(expr)                                                   \
  do {                                                                 \
    hipError_t _e = (expr);                                            \
    if (_e != hipSuccess) return fail(#expr, hipGetErrorString(_e));   \
  } while (0)
#define ORCCHK(expr)               \
  do {                             \
    int _r = (expr);               \
    if (_r != 0) return _r;        \
  } while (0)

namespace {

struct Raw {
  bf16_t* p = nullptr;
  std::vector<int64_t> shape;
  size_t numel = 0;
};
struct Packed {
  bf16_t* p = nullptr;
  int N = 0, K = 0, Nvalid = 0;   // padded rows / cols, valid rows
  // lossless 12-bit copy for the decode GEMVs (gemv.hip); null = the GEMV streams p
  uint8_t* wc = nullptr; uint8_t* emin = nullptr; uint16_t* patch = nullptr;
  int wc_group = 0;   // block order inside wc (GemvArgs::wc_group): ORC_DECODE_LAYOUT=rowmajor keeps 0, default kCwGroup
};
struct ClipLayer {
  bf16_t *ln1w, *ln1b, *ln2w, *ln2b, *bqkv, *bo, *b1, *b2;
  Packed qkv, o, fc1, fc2;
};
struct PoolLayer {
  bf16_t *bqkv, *bo, *ln1w, *ln1b, *bi, *bout, *ln2w, *ln2b;
  Packed qkv, o, wi, wout;
};
struct LlamaLayer {
  bf16_t *ln_in, *ln_post;
  Packed qkv, qkv_dec, o, gu, gu_dec, down;   // *_dec: decode copies with the preceding RMSNorm weight folded into the columns
};

static inline int round_up(int x, int m) { return (x + m - 1) / m * m; }

// A launch has at most kMaxRows = 32 ROWS (two MFMA B-operand tiles of 16 in the decode GEMVs; the prefill batches the same
// way); the KV cache and the greedy state have up to kMaxSlots SLOTS, so that frames can wait prefilled while others decode.
constexpr int kMaxSlots = 64;
// dev_ints layout (ints): 16 header, per-slot state arrays of kMaxSlots each, three per-launch-row arrays of kMaxRows, then
// tokens [slots][max_new_tokens]
enum { DI_UNF = 16, DI_NEXT = DI_UNF + kMaxSlots, DI_ARGMAX = DI_NEXT + kMaxSlots, DI_KBEG = DI_ARGMAX + kMaxSlots,
       DI_CURLEN = DI_KBEG + kMaxSlots, DI_ROWSTEP = DI_CURLEN + kMaxSlots, DI_LIMIT = DI_ROWSTEP + kMaxSlots,
       DI_KEND = DI_LIMIT + kMaxSlots, DI_ROWOFF = DI_KEND + kMaxRows, DI_ROWVALID = DI_ROWOFF + kMaxRows,
       DI_TOKENS = DI_ROWVALID + kMaxRows };

}  // namespace

struct orc_engine {
  orc_config c;
  bool finalized = false;
  std::map<std::string, Raw> raw;
  std::vector<void*> owned;   // device allocations freed at destroy

  // CLIP
  Packed patch_w;
  bf16_t *clip_cls = nullptr, *clip_pos = nullptr, *pre_lnw = nullptr, *pre_lnb = nullptr, *post_lnw = nullptr, *post_lnb = nullptr;
  std::vector<ClipLayer> clip;
  // pooler
  bf16_t *pool_tt0 = nullptr, *pool_pos = nullptr, *pool_elnw = nullptr, *pool_elnb = nullptr;
  std::vector<PoolLayer> pool;
  // projector
  Packed proj0, proj2;
  bf16_t *proj_b0 = nullptr, *proj_b2 = nullptr;
  // llama
  bf16_t* embed = nullptr;
  std::vector<LlamaLayer> llama;
  bf16_t* final_norm = nullptr;
  Packed lm_head, lm_head_dec;
  bf16_t *cos_tab = nullptr, *sin_tab = nullptr;
  int maxpos = 0;

  // KV cache: per layer K and V, [B][H][Tmax][128]
  bf16_t *kcache = nullptr, *vcache = nullptr;
  size_t kv_layer_elems = 0;
  long c_bs = 0, c_hs = 0;

  // workspace
  int ws_rows = 0;
  bf16_t *w_h = nullptr, *w_xn = nullptr, *w_qkv = nullptr, *w_att = nullptr, *w_mlp = nullptr, *w_aux = nullptr;
  float* w_logits = nullptr;
  float* w_part = nullptr;
  float* d_ssq = nullptr;   // [16][d_model/16] per-n-tile sums of squares of the decode hidden state
  // per decode ROW, refreshed by the token gather of every step (kernels.h RowMetaArgs): {slot, cached keys, left pad, unfinished},
  // and the rotary table rows of the row's position -- what the q/k/v epilogue otherwise chases through three dependent loads
  int* d_rowmeta = nullptr; bf16_t* d_rowcos = nullptr; bf16_t* d_rowsin = nullptr;
  bf16_t* d_hxf = nullptr;   // decode hidden rows in the fragment-ordered layout (input of the norm-folded projections)
  bf16_t *d_h = nullptr, *d_xn = nullptr, *d_qkv = nullptr, *d_att = nullptr, *d_mlp = nullptr;   // decode (<=16 rows)
  int *dev_ints = nullptr;   // [0]=step [2]=n_unfinished, then per-row arrays of 16 (DI_* offsets), then the token buffer
  int *d_step, *d_nunf, *d_unf, *d_next, *d_argmax, *d_kbeg, *d_kend, *d_rowoff, *d_rowvalid, *d_curlen, *d_rowstep, *d_limit, *d_tokens;
  int32_t* d_plan = nullptr; // tile list of a packed prefill's attention
  int* d_pfkbeg = nullptr;   // [16] left pad of the rows of the prefill being launched (attention reads it per launch row)
  bool compress_decode = true;   // ORC_DECODE_WEIGHTS=plain turns the 12-bit decode copies off (A/B runs)
  // ORC_DECODE_NORM=exact: the decode path runs every RMSNorm as its own launch with the reference's rounding points (fp32
  // statistics, bf16(x * r) * w: the prefill's kernel) in front of un-folded decode weight copies, instead of folding the norm
  // weight into the projection and the row scale into its epilogue (A/B switch for the folded norm's changed rounding points)
  bool fold_norm = true;
  // bookkeeping of the 12-bit copies (orc_decode_weight_stats): decode matrices seen / compressed, their elements and escapes
  int64_t cw_mats = 0, cw_done = 0, cw_elems = 0, cw_escapes = 0, cw_flagged_blocks = 0, cw_blocks = 0;
  bool stream_mode = false;  // continuous batching (orc_stream_begin): decode rows are re-pointed at slots prefilled ahead
  RowMap row_map;            // decode row -> slot (host copy; goes to the kernels by value)
  int cur_batch = 0, cur_T = 0;
  int steps_issued = 0;   // decode steps enqueued since the last prefill (host-side mirror of the device cur_len - T)
  // sampled HIP-event timing of the dominant decode kernel (gate/up GEMV), see orc_profile_*
  bool prof_on = false;
  std::vector<hipEvent_t> ev_a, ev_b;
  int ev_used = 0;

  int alloc(void** p, size_t bytes) {
    hipError_t e = hipMalloc(p, bytes ? bytes : 16);
    if (e != hipSuccess) return fail("hipMalloc", hipGetErrorString(e));
    owned.push_back(*p);
    return 0;
  }
};

namespace {

int get_raw(orc_engine* e, const std::string& name, Raw** out, bool required = true) {
  auto it = e->raw.find(name);
  if (it == e->raw.end()) {
    *out = nullptr;
    if (required) return fail("missing weight", name.c_str());
    return 0;
  }
  *out = &it->second;
  return 0;
}

// take ownership of a raw tensor as-is (1-D params, embeddings)
int take(orc_engine* e, const std::string& name, bf16_t** dst, size_t expect_numel) {
  Raw* r;
  ORCCHK(get_raw(e, name, &r));
  if (r->numel != expect_numel) return fail("bad weight size", name.c_str());
  *dst = r->p;
  r->p = nullptr;   // ownership stays in e->owned
  return 0;
}

// concatenate row-major matrices along rows into a temp, pack, free the temp
int pack_rows(orc_engine* e, const std::vector<std::string>& names, int K, const std::vector<int>* rowmap_host, int align_n,
              Packed* out, const bf16_t* colscale = nullptr) {
  int nsrc = 0;
  std::vector<Raw*> rs;
  for (auto& n : names) {
    Raw* r;
    ORCCHK(get_raw(e, n, &r));
    if (r->shape.size() < 2) return fail("weight is not a matrix", n.c_str());
    int64_t cols = 1;
    for (size_t i = 1; i < r->shape.size(); ++i) cols *= r->shape[i];
    if (cols != K) return fail("bad weight inner size", n.c_str());
    nsrc += (int)r->shape[0];
    rs.push_back(r);
  }
  bf16_t* tmp = nullptr;
  const bf16_t* src = rs[0]->p;
  if (rs.size() > 1) {
    HIPCHK(hipMalloc((void**)&tmp, (size_t)nsrc * K * 2));
    size_t off = 0;
    for (auto* r : rs) {
      HIPCHK(hipMemcpy(tmp + off, r->p, r->numel * 2, hipMemcpyDeviceToDevice));
      off += r->numel;
    }
    src = tmp;
  }
  const int nrows = rowmap_host ? (int)rowmap_host->size() : nsrc;
  const int Np = round_up(nrows, align_n), Kp = round_up(K, 64);
  int* rm = nullptr;
  if (rowmap_host) {
    std::vector<int> full(Np, -1);
    memcpy(full.data(), rowmap_host->data(), rowmap_host->size() * sizeof(int));
    HIPCHK(hipMalloc((void**)&rm, Np * sizeof(int)));
    HIPCHK(hipMemcpy(rm, full.data(), Np * sizeof(int), hipMemcpyHostToDevice));
  }
  bf16_t* wp;
  ORCCHK(e->alloc((void**)&wp, (size_t)Np * Kp * 2));
  HIPCHK(launch_pack_weight(src, nsrc, K, rm, wp, Np, Kp, 0, colscale));
  HIPCHK(hipDeviceSynchronize());
  if (tmp) HIPCHK(hipFree(tmp));
  if (rm) HIPCHK(hipFree(rm));
  out->p = wp; out->N = Np; out->K = Kp; out->Nvalid = nrows;
  return 0;
}

int concat_vec(orc_engine* e, const std::vector<std::string>& names, bf16_t** dst, int pad_to) {
  size_t tot = 0;
  std::vector<Raw*> rs;
  for (auto& n : names) {
    Raw* r;
    ORCCHK(get_raw(e, n, &r));
    rs.push_back(r);
    tot += r->numel;
  }
  size_t padded = round_up((int)tot, pad_to);
  ORCCHK(e->alloc((void**)dst, padded * 2));
  HIPCHK(hipMemset(*dst, 0, padded * 2));
  size_t off = 0;
  for (auto* r : rs) {
    HIPCHK(hipMemcpy(*dst + off, r->p, r->numel * 2, hipMemcpyDeviceToDevice));
    off += r->numel;
  }
  return 0;
}

void free_raw(orc_engine* e, const std::vector<std::string>& names) {
  for (auto& n : names) {
    auto it = e->raw.find(n);
    if (it == e->raw.end() || !it->second.p) continue;
    void* p = it->second.p;
    for (auto& o : e->owned)
      if (o == p) { o = nullptr; break; }
    (void)hipFree(p);
    it->second.p = nullptr;
  }
}

inline hipStream_t S(void* s) { return (hipStream_t)s; }

int gemm(const bf16_t* X, int ldx, const Packed& W, const bf16_t* bias, const bf16_t* R, int ldr, void* C, int ldc, int M,
         int epi, hipStream_t s, bool small) {
  GemmArgs a;
  a.X = X; a.ldx = ldx; a.Wp = W.p; a.bias = bias; a.R = R; a.ldr = ldr; a.C = C; a.ldc = ldc;
  a.M = M; a.N = W.N; a.K = W.K;
  a.Nvalid = (epi == EPI_SWIGLU) ? W.Nvalid / 2 : W.Nvalid;
  hipError_t err = small ? launch_gemv(a, epi, s) : launch_gemm(a, epi, s);
  if (err != hipSuccess) return fail(small ? "launch_gemv" : "launch_gemm", hipGetErrorString(err));
  return 0;
}

void free_owned(orc_engine* e, void* p) {
  if (!p) return;
  for (auto& o : e->owned)
    if (o == p) { (void)hipFree(o); o = nullptr; }
}

// Decode GEMVs are HBM-bound on the weight stream and their vector ALUs idle: give W a lossless 12-bit copy (768 B per 1-KiB
// fragment block, bit-exact decode in the kernel, gemv.hip) that the decode launches stream instead. epi = the epilogue the
// decode GEMV of this matrix runs with (it fixes the unit size of the patch tables). drop_plain: the bf16 copy is used by
// nothing else (the norm-folded decode copies) and is freed. A matrix with a unit of more than 254 non-zero out-of-range elements
// keeps its bf16 stream (25 % more bytes for that matrix): LOUDLY -- one stderr line per matrix here, a summary line at
// orc_engine_finalize, and the counts through orc_decode_weight_stats (r2 kept it silent).
int compress_for_decode(orc_engine* e, Packed* W, int epi, bool drop_plain, const char* what = "") {
  if (!W->p) return 0;
  ++e->cw_mats;
  e->cw_elems += (int64_t)W->N * W->K;
  e->cw_blocks += (int64_t)(W->N / 16) * (W->K / 32);
  if (!e->compress_decode) return 0;
  const int nt_unit = gemv_unit_tiles(epi, W->N);
  const size_t nblk = (size_t)(W->N / 16) * (W->K / 32);
  const int units = W->N / 16 / nt_unit;
  uint8_t *wc = nullptr, *em = nullptr;
  uint16_t* patch = nullptr;
  int* cnt = nullptr;
  ORCCHK(e->alloc((void**)&wc, nblk * 768));
  ORCCHK(e->alloc((void**)&em, (nblk + 7) & ~(size_t)3));
  ORCCHK(e->alloc((void**)&patch, (size_t)units * 256 * 2));
  HIPCHK(hipMalloc((void**)&cnt, (size_t)(units + 1) * 4));
  HIPCHK(hipMemset(cnt + units, 0, 4));
  static const int group = []() { const char* l = getenv("ORC_DECODE_LAYOUT"); return l && strcmp(l, "rowmajor") == 0 ? 0 : kCwGroup; }();
  HIPCHK(launch_compress_weight(W->p, W->N, W->K, nt_unit, wc, em, patch, cnt, cnt + units, 0, group));
  W->wc_group = group;
  std::vector<int> hc(units + 1);
  HIPCHK(hipMemcpy(hc.data(), cnt, (size_t)(units + 1) * 4, hipMemcpyDeviceToHost));
  HIPCHK(hipFree(cnt));
  const int overflow = hc[units];
  int64_t esc = 0;
  int worst = 0;
  for (int u = 0; u < units; ++u) { esc += hc[u]; worst = hc[u] > worst ? hc[u] : worst; }
  if (overflow) {
    fprintf(stderr, "[oracle_hip] decode weights %s (%d x %d): a %d-tile unit has %d out-of-range elements (> 254 patch entries): "
            "this matrix keeps its bf16 stream (+33 %% bytes per decode step for it)\n", what, W->N, W->K, nt_unit, worst);
    free_owned(e, wc); free_owned(e, em); free_owned(e, patch);
    return 0;
  }
  {   // flagged blocks (their decode takes the patch-table path): counted on the host from the side bytes
    std::vector<uint8_t> he(nblk);
    HIPCHK(hipMemcpy(he.data(), em, nblk, hipMemcpyDeviceToHost));
    int64_t fl = 0;
    for (size_t i = 0; i < nblk; ++i) fl += he[i] >> 7;
    e->cw_flagged_blocks += fl;
  }
  ++e->cw_done;
  e->cw_escapes += esc;
  W->wc = wc; W->emin = em; W->patch = patch;
  if (drop_plain) { free_owned(e, W->p); W->p = nullptr; }
  return 0;
}

}  // namespace

// ============================================================================ lifecycle
extern "C" int orc_engine_create(const orc_config* cfg, orc_engine** out) {
  if (!cfg || !out) return fail("orc_engine_create", "null argument");
  const orc_config& c = *cfg;
  if (c.n_heads <= 0 || c.d_model != c.n_heads * 128) return fail("orc_engine_create", "LLaMA head_dim must be 128");
  if (c.clip_d % c.clip_heads || c.clip_d / c.clip_heads != 64) return fail("orc_engine_create", "CLIP head_dim must be 64");
  if (c.clip_d / c.pool_heads != 128) return fail("orc_engine_create", "pooler head_dim must be 128");
  if (c.max_batch < 1 || c.max_batch > kMaxSlots) return fail("orc_engine_create", "max_batch (KV-cache slots) must be in 1..64");
  if (c.d_model % 256 || c.d_ff % 64 || c.vocab % 128 || c.clip_d % 128 || c.clip_ff % 128 || c.pool_ff % 128)
    return fail("orc_engine_create", "widths must be multiples of 128 (d_model: 256, i.e. an even head count; d_ff: 64)");
  if (c.d_model > 4096) return fail("orc_engine_create", "d_model above 4096 is not supported (decode row-scale partials: d_model / 16 <= 256)");
  if (c.max_seq < 2 || c.max_new_tokens < 1 || c.max_images < 1) return fail("orc_engine_create", "capacities must be positive");
  if (c.clip_image % c.clip_patch) return fail("orc_engine_create", "image size not a multiple of the patch size");
  orc_engine* e = new orc_engine();
  e->c = c;
  *out = e;
  return 0;
}

extern "C" void orc_engine_destroy(orc_engine* e) {
  if (!e) return;
  (void)hipDeviceSynchronize();
  for (void* p : e->owned)
    if (p) (void)hipFree(p);
  delete e;
}

extern "C" int orc_engine_load_weight(orc_engine* e, const char* name, const void* data, int on_device,
                                      const int64_t* shape, int ndim) {
  if (!e || !name || !data || !shape || ndim < 1) return fail("orc_engine_load_weight", "bad argument");
  if (e->finalized) return fail("orc_engine_load_weight", "engine already finalized");
  Raw r;
  r.numel = 1;
  for (int i = 0; i < ndim; ++i) {
    r.shape.push_back(shape[i]);
    r.numel *= (size_t)shape[i];
  }
  ORCCHK(e->alloc((void**)&r.p, r.numel * 2));
  HIPCHK(hipMemcpy(r.p, data, r.numel * 2, on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice));
  auto old = e->raw.find(name);
  if (old != e->raw.end()) free_raw(e, {name});
  e->raw[name] = r;
  return 0;
}

extern "C" int orc_engine_finalize(orc_engine* e) {
  if (!e) return fail("orc_engine_finalize", "null engine");
  if (e->finalized) return 0;
  const orc_config& c = e->c;
  char buf[256];
  // ---------------- CLIP
  {
    const std::string p = "model.vision_tower.vision_tower.vision_model.";
    const int kpatch = 3 * c.clip_patch * c.clip_patch;
    ORCCHK(pack_rows(e, {p + "embeddings.patch_embedding.weight"}, kpatch, nullptr, 256, &e->patch_w));
    free_raw(e, {p + "embeddings.patch_embedding.weight"});
    const int tokens = (c.clip_image / c.clip_patch) * (c.clip_image / c.clip_patch) + 1;
    ORCCHK(take(e, p + "embeddings.class_embedding", &e->clip_cls, c.clip_d));
    ORCCHK(take(e, p + "embeddings.position_embedding.weight", &e->clip_pos, (size_t)tokens * c.clip_d));
    ORCCHK(take(e, p + "pre_layrnorm.weight", &e->pre_lnw, c.clip_d));
    ORCCHK(take(e, p + "pre_layrnorm.bias", &e->pre_lnb, c.clip_d));
    ORCCHK(take(e, p + "post_layernorm.weight", &e->post_lnw, c.clip_d));
    ORCCHK(take(e, p + "post_layernorm.bias", &e->post_lnb, c.clip_d));
    e->clip.resize(c.clip_layers);
    for (int i = 0; i < c.clip_layers; ++i) {
      snprintf(buf, sizeof(buf), "%sencoder.layers.%d.", p.c_str(), i);
      const std::string q = buf;
      ClipLayer& L = e->clip[i];
      ORCCHK(take(e, q + "layer_norm1.weight", &L.ln1w, c.clip_d));
      ORCCHK(take(e, q + "layer_norm1.bias", &L.ln1b, c.clip_d));
      ORCCHK(take(e, q + "layer_norm2.weight", &L.ln2w, c.clip_d));
      ORCCHK(take(e, q + "layer_norm2.bias", &L.ln2b, c.clip_d));
      std::vector<std::string> w3 = {q + "self_attn.q_proj.weight", q + "self_attn.k_proj.weight", q + "self_attn.v_proj.weight"};
      ORCCHK(pack_rows(e, w3, c.clip_d, nullptr, 256, &L.qkv));
      ORCCHK(concat_vec(e, {q + "self_attn.q_proj.bias", q + "self_attn.k_proj.bias", q + "self_attn.v_proj.bias"}, &L.bqkv, 128));
      ORCCHK(pack_rows(e, {q + "self_attn.out_proj.weight"}, c.clip_d, nullptr, 256, &L.o));
      ORCCHK(take(e, q + "self_attn.out_proj.bias", &L.bo, c.clip_d));
      ORCCHK(pack_rows(e, {q + "mlp.fc1.weight"}, c.clip_d, nullptr, 256, &L.fc1));
      ORCCHK(take(e, q + "mlp.fc1.bias", &L.b1, c.clip_ff));
      ORCCHK(pack_rows(e, {q + "mlp.fc2.weight"}, c.clip_ff, nullptr, 256, &L.fc2));
      ORCCHK(take(e, q + "mlp.fc2.bias", &L.b2, c.clip_d));
      w3.push_back(q + "self_attn.out_proj.weight");
      w3.push_back(q + "mlp.fc1.weight");
      w3.push_back(q + "mlp.fc2.weight");
      w3.push_back(q + "self_attn.q_proj.bias");
      w3.push_back(q + "self_attn.k_proj.bias");
      w3.push_back(q + "self_attn.v_proj.bias");
      free_raw(e, w3);
    }
  }
  // ---------------- pooler
  {
    const std::string p = "model.image_pooler.bert.";
    Raw* r;
    ORCCHK(get_raw(e, p + "embeddings.token_type_embeddings.weight", &r));
    if (r->numel < (size_t)c.clip_d) return fail("bad weight size", "token_type_embeddings");
    e->pool_tt0 = r->p;   // row 0
    r->p = nullptr;
    ORCCHK(take(e, p + "embeddings.position_embeddings.weight", &e->pool_pos, (size_t)c.pool_maxpos * c.clip_d));
    ORCCHK(take(e, p + "embeddings.LayerNorm.weight", &e->pool_elnw, c.clip_d));
    ORCCHK(take(e, p + "embeddings.LayerNorm.bias", &e->pool_elnb, c.clip_d));
    e->pool.resize(c.pool_layers);
    for (int i = 0; i < c.pool_layers; ++i) {
      snprintf(buf, sizeof(buf), "%sencoder.layer.%d.", p.c_str(), i);
      const std::string q = buf;
      PoolLayer& L = e->pool[i];
      std::vector<std::string> w3 = {q + "attention.self.query.weight", q + "attention.self.key.weight", q + "attention.self.value.weight"};
      ORCCHK(pack_rows(e, w3, c.clip_d, nullptr, 256, &L.qkv));
      ORCCHK(concat_vec(e, {q + "attention.self.query.bias", q + "attention.self.key.bias", q + "attention.self.value.bias"}, &L.bqkv, 128));
      ORCCHK(pack_rows(e, {q + "attention.output.dense.weight"}, c.clip_d, nullptr, 256, &L.o));
      ORCCHK(take(e, q + "attention.output.dense.bias", &L.bo, c.clip_d));
      ORCCHK(take(e, q + "attention.output.LayerNorm.weight", &L.ln1w, c.clip_d));
      ORCCHK(take(e, q + "attention.output.LayerNorm.bias", &L.ln1b, c.clip_d));
      ORCCHK(pack_rows(e, {q + "intermediate.dense.weight"}, c.clip_d, nullptr, 256, &L.wi));
      ORCCHK(take(e, q + "intermediate.dense.bias", &L.bi, c.pool_ff));
      ORCCHK(pack_rows(e, {q + "output.dense.weight"}, c.pool_ff, nullptr, 256, &L.wout));
      ORCCHK(take(e, q + "output.dense.bias", &L.bout, c.clip_d));
      ORCCHK(take(e, q + "output.LayerNorm.weight", &L.ln2w, c.clip_d));
      ORCCHK(take(e, q + "output.LayerNorm.bias", &L.ln2b, c.clip_d));
      w3.push_back(q + "attention.output.dense.weight");
      w3.push_back(q + "intermediate.dense.weight");
      w3.push_back(q + "output.dense.weight");
      w3.push_back(q + "attention.self.query.bias");
      w3.push_back(q + "attention.self.key.bias");
      w3.push_back(q + "attention.self.value.bias");
      free_raw(e, w3);
    }
  }
  // ---------------- projector
  ORCCHK(pack_rows(e, {"model.mm_projector.0.weight"}, c.clip_d, nullptr, 256, &e->proj0));
  ORCCHK(take(e, "model.mm_projector.0.bias", &e->proj_b0, c.d_model));
  ORCCHK(pack_rows(e, {"model.mm_projector.2.weight"}, c.d_model, nullptr, 256, &e->proj2));
  ORCCHK(take(e, "model.mm_projector.2.bias", &e->proj_b2, c.d_model));
  free_raw(e, {"model.mm_projector.0.weight", "model.mm_projector.2.weight"});
  // ---------------- LLaMA
  ORCCHK(take(e, "model.embed_tokens.weight", &e->embed, (size_t)c.vocab * c.d_model));
  ORCCHK(take(e, "model.norm.weight", &e->final_norm, c.d_model));
  ORCCHK(pack_rows(e, {"lm_head.weight"}, c.d_model, nullptr, 256, &e->lm_head));
  {
    const char* nm = getenv("ORC_DECODE_NORM");
    e->fold_norm = !(nm && strcmp(nm, "exact") == 0);
  }
  ORCCHK(pack_rows(e, {"lm_head.weight"}, c.d_model, nullptr, 256, &e->lm_head_dec, e->fold_norm ? e->final_norm : nullptr));
  free_raw(e, {"lm_head.weight"});
  {
    const char* m = getenv("ORC_DECODE_WEIGHTS");
    e->compress_decode = !(m && strcmp(m, "plain") == 0);
    const char* nm = getenv("ORC_DECODE_NORM");
    e->fold_norm = !(nm && strcmp(nm, "exact") == 0);
  }
  ORCCHK(compress_for_decode(e, &e->lm_head_dec, EPI_F32, true, "lm_head"));
  e->llama.resize(c.n_layers);
  std::vector<int> gu_map(2 * c.d_ff);
  for (int pr = 0; pr < 2 * c.d_ff; ++pr) {
    const int t = pr / 32, wi = pr % 32;   // gate tile, up tile alternate every 16 rows
    gu_map[pr] = wi < 16 ? 16 * t + wi : c.d_ff + 16 * t + (wi - 16);
  }
  // decode copy of the fused q/k/v weight, in units of three 16-row tiles: tile j and tile j+4 of a q or k head (so one
  // workgroup of the decode GEMV holds a head dim and its rotary partner (d, d+64) in the same lane) followed by one tile
  // of the v projection. There are 8 * n_heads rotary pairs and as many v tiles: d_model / 16 units of equal work (256 for
  // the 7B model: one workgroup per CU), unit u = pair u of the q|k sections + v rows [16u, 16u + 16).
  std::vector<int> qkv_dec_map(3 * c.d_model);
  for (int pr = 0; pr < 3 * c.d_model; ++pr) {
    const int unit = pr / 48, tile = (pr % 48) / 16, rr = pr % 16, hs = unit / 4, j = unit % 4;
    qkv_dec_map[pr] = tile < 2 ? hs * 128 + (j + 4 * tile) * 16 + rr : 2 * c.d_model + unit * 16 + rr;
  }
  for (int i = 0; i < c.n_layers; ++i) {
    snprintf(buf, sizeof(buf), "model.layers.%d.", i);
    const std::string q = buf;
    LlamaLayer& L = e->llama[i];
    ORCCHK(take(e, q + "input_layernorm.weight", &L.ln_in, c.d_model));
    ORCCHK(take(e, q + "post_attention_layernorm.weight", &L.ln_post, c.d_model));
    std::vector<std::string> w3 = {q + "self_attn.q_proj.weight", q + "self_attn.k_proj.weight", q + "self_attn.v_proj.weight"};
    ORCCHK(pack_rows(e, w3, c.d_model, nullptr, 256, &L.qkv));
    ORCCHK(pack_rows(e, w3, c.d_model, &qkv_dec_map, 256, &L.qkv_dec, e->fold_norm ? L.ln_in : nullptr));
    ORCCHK(pack_rows(e, {q + "self_attn.o_proj.weight"}, c.d_model, nullptr, 256, &L.o));
    std::vector<std::string> w2 = {q + "mlp.gate_proj.weight", q + "mlp.up_proj.weight"};
    ORCCHK(pack_rows(e, w2, c.d_model, &gu_map, 256, &L.gu));
    ORCCHK(pack_rows(e, w2, c.d_model, &gu_map, 256, &L.gu_dec, e->fold_norm ? L.ln_post : nullptr));
    ORCCHK(pack_rows(e, {q + "mlp.down_proj.weight"}, c.d_ff, nullptr, 256, &L.down));
    ORCCHK(compress_for_decode(e, &L.qkv_dec, EPI_ROPE_KV, true, (q + "self_attn.{q,k,v}_proj").c_str()));
    ORCCHK(compress_for_decode(e, &L.gu_dec, EPI_SWIGLU, true, (q + "mlp.{gate,up}_proj").c_str()));
    ORCCHK(compress_for_decode(e, &L.o, EPI_RESIDUAL, false, (q + "self_attn.o_proj").c_str()));      // the prefill GEMM keeps reading the bf16 copy
    ORCCHK(compress_for_decode(e, &L.down, EPI_RESIDUAL, false, (q + "mlp.down_proj").c_str()));
    w3.push_back(q + "self_attn.o_proj.weight");
    w3.push_back(w2[0]);
    w3.push_back(w2[1]);
    w3.push_back(q + "mlp.down_proj.weight");
    free_raw(e, w3);
  }
  // ---------------- rotary tables: cos/sin(fp32 angle) rounded to bf16 (transformers LlamaRotaryEmbedding)
  {
    e->maxpos = c.max_seq + 8;
    std::vector<bf16_t> ct((size_t)e->maxpos * 64), st((size_t)e->maxpos * 64);
    for (int i = 0; i < 64; ++i) {
      const float expo = (float)(2 * i) / 128.0f;
      const float inv = 1.0f / powf(c.rope_theta, expo);
      for (int p = 0; p < e->maxpos; ++p) {
        const float ang = inv * (float)p;
        const float cf = (float)cos((double)ang), sf = (float)sin((double)ang);
        uint32_t u;
        memcpy(&u, &cf, 4);
        ct[(size_t)p * 64 + i] = (bf16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
        memcpy(&u, &sf, 4);
        st[(size_t)p * 64 + i] = (bf16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
      }
    }
    ORCCHK(e->alloc((void**)&e->cos_tab, ct.size() * 2));
    ORCCHK(e->alloc((void**)&e->sin_tab, st.size() * 2));
    HIPCHK(hipMemcpy(e->cos_tab, ct.data(), ct.size() * 2, hipMemcpyHostToDevice));
    HIPCHK(hipMemcpy(e->sin_tab, st.data(), st.size() * 2, hipMemcpyHostToDevice));
  }
  // ---------------- KV cache + workspace
  {
    // (slot, head) regions of max_seq keys x 256 B. The (row, head) workgroups of the decode attention walk their regions in step, so a
    // region stride that is a multiple of 64 KiB (max_seq a multiple of 256: 1024, 2048, the builder's 4096) keeps them on the same HBM
    // channels (measured: max_seq 1024 decodes 1.3 % slower than 992 or 1056); such lengths get 32 keys (8 KiB) of padding per region.
    const int kv_pad = (c.max_seq % 256 == 0) ? 32 : 0;
    e->c_hs = (long)(c.max_seq + kv_pad) * 128;
    e->c_bs = e->c_hs * c.n_heads;
    e->kv_layer_elems = (size_t)e->c_bs * c.max_batch;
    ORCCHK(e->alloc((void**)&e->kcache, e->kv_layer_elems * c.n_layers * 2));
    ORCCHK(e->alloc((void**)&e->vcache, e->kv_layer_elems * c.n_layers * 2));
    const int tokens = (c.clip_image / c.clip_patch) * (c.clip_image / c.clip_patch) + 1;
    int rows = c.max_images * tokens;
    const int max_rows = c.max_batch < kMaxRows ? c.max_batch : kMaxRows;   // rows of one prefill / pooler / decode launch
    if (max_rows * c.max_seq > rows) rows = max_rows * c.max_seq;
    if (max_rows * c.pool_maxpos > rows) rows = max_rows * c.pool_maxpos;
    rows = round_up(rows, 128);
    e->ws_rows = rows;
    const int wd = c.d_model > c.clip_d ? c.d_model : c.clip_d;
    int wm = c.d_ff;
    if (c.clip_ff > wm) wm = c.clip_ff;
    if (c.pool_ff > wm) wm = c.pool_ff;
    if (c.d_model > wm) wm = c.d_model;
    ORCCHK(e->alloc((void**)&e->w_h, (size_t)rows * wd * 2));
    ORCCHK(e->alloc((void**)&e->w_xn, (size_t)rows * wd * 2));
    ORCCHK(e->alloc((void**)&e->w_att, (size_t)rows * wd * 2));
    ORCCHK(e->alloc((void**)&e->w_aux, (size_t)rows * wd * 2));
    ORCCHK(e->alloc((void**)&e->w_qkv, (size_t)rows * wd * 3 * 2));
    ORCCHK(e->alloc((void**)&e->w_mlp, (size_t)rows * wm * 2));
    ORCCHK(e->alloc((void**)&e->w_logits, (size_t)kMaxRows * c.vocab * 4));
    ORCCHK(e->alloc((void**)&e->w_part, (size_t)kMaxRows * c.n_heads * DECODE_NSPLIT * 130 * 4));
    ORCCHK(e->alloc((void**)&e->d_plan, (size_t)attn_plan_ints(rows) * 4));
    ORCCHK(e->alloc((void**)&e->d_ssq, (size_t)kMaxRows * (c.d_model / 16) * 4));
    ORCCHK(e->alloc((void**)&e->d_rowmeta, (size_t)kMaxRows * 4 * 4));
    ORCCHK(e->alloc((void**)&e->d_rowcos, (size_t)kMaxRows * 64 * 2));
    ORCCHK(e->alloc((void**)&e->d_rowsin, (size_t)kMaxRows * 64 * 2));
    ORCCHK(e->alloc((void**)&e->d_h, (size_t)kMaxRows * c.d_model * 2));
    ORCCHK(e->alloc((void**)&e->d_hxf, (size_t)kMaxRows * c.d_model * 2));
    HIPCHK(hipMemset(e->d_hxf, 0, (size_t)kMaxRows * c.d_model * 2));
    ORCCHK(e->alloc((void**)&e->d_xn, (size_t)kMaxRows * c.d_model * 2));
    ORCCHK(e->alloc((void**)&e->d_att, (size_t)kMaxRows * c.d_model * 2));
    ORCCHK(e->alloc((void**)&e->d_qkv, (size_t)kMaxRows * c.d_model * 3 * 2));
    ORCCHK(e->alloc((void**)&e->d_mlp, (size_t)kMaxRows * c.d_ff * 2));
    const size_t nint = DI_TOKENS + (size_t)kMaxSlots * c.max_new_tokens;
    ORCCHK(e->alloc((void**)&e->dev_ints, nint * 4));
    HIPCHK(hipMemset(e->dev_ints, 0, nint * 4));
    int* di = e->dev_ints;
    e->d_step = di;
    e->d_nunf = di + 2;
    e->d_unf = di + DI_UNF; e->d_next = di + DI_NEXT; e->d_argmax = di + DI_ARGMAX; e->d_kbeg = di + DI_KBEG;
    e->d_kend = di + DI_KEND; e->d_rowoff = di + DI_ROWOFF; e->d_rowvalid = di + DI_ROWVALID;
    e->d_curlen = di + DI_CURLEN; e->d_rowstep = di + DI_ROWSTEP; e->d_limit = di + DI_LIMIT;
    e->d_tokens = di + DI_TOKENS;
    e->d_pfkbeg = di + DI_KEND;   // (the pooler's key-end array is not used by a LLaMA prefill)
    e->row_map = identity_map();
  }
  HIPCHK(hipDeviceSynchronize());
  if (e->compress_decode && e->cw_done < e->cw_mats)
    fprintf(stderr, "[oracle_hip] %lld of %lld decode weight matrices could not take the lossless 12-bit stream and stay bf16 "
            "(orc_decode_weight_stats / orc_decode_stream_bytes report it)\n", (long long)(e->cw_mats - e->cw_done), (long long)e->cw_mats);
  e->finalized = true;
  return 0;
}

// ============================================================================ vision
static int clip_forward(orc_engine* e, const void* images, int n, int n_layers, hipStream_t s) {
  const orc_config& c = e->c;
  const int G = c.clip_image / c.clip_patch, patches = G * G, tokens = patches + 1, d = c.clip_d;
  if (n <= 0 || n > c.max_images) return fail("vision", "n_images outside 1..max_images");
  const int Mp = n * patches, M = n * tokens;
  // patch embedding as GEMM: im2col -> [Mp][Kp] x W[d][Kp]
  HIPCHK(launch_im2col((const bf16_t*)images, n, c.clip_image, c.clip_patch, e->w_mlp, e->patch_w.K, s));
  ORCCHK(gemm(e->w_mlp, e->patch_w.K, e->patch_w, nullptr, nullptr, 0, e->w_xn, d, Mp, EPI_NONE, s, false));
  HIPCHK(launch_clip_embed(e->w_xn, e->clip_cls, e->clip_pos, nullptr, nullptr, e->w_h, n, tokens, d, 0.f, s));
  HIPCHK(launch_layernorm(e->w_h, d, e->pre_lnw, e->pre_lnb, e->w_h, d, M, d, c.clip_eps, s));
  for (int i = 0; i < n_layers; ++i) {
    const ClipLayer& L = e->clip[i];
    HIPCHK(launch_layernorm(e->w_h, d, L.ln1w, L.ln1b, e->w_xn, d, M, d, c.clip_eps, s));
    ORCCHK(gemm(e->w_xn, d, L.qkv, L.bqkv, nullptr, 0, e->w_qkv, 3 * d, M, EPI_NONE, s, false));
    AttnArgs a;
    a.Q = e->w_qkv; a.K = e->w_qkv + d; a.V = e->w_qkv + 2 * d;
    a.q_bs = a.k_bs = a.v_bs = (long)tokens * 3 * d; a.q_hs = a.k_hs = a.v_hs = 64; a.q_ts = a.k_ts = a.v_ts = 3 * d;
    a.O = e->w_att; a.o_bs = (long)tokens * d; a.o_hs = 64; a.o_ts = d;
    a.B = n; a.H = c.clip_heads; a.Sq = tokens; a.Sk = tokens; a.kbeg = nullptr; a.kend = nullptr; a.causal = 0; a.q_off = 0;
    a.scale = 0.125f;   // 64^-0.5
    HIPCHK(launch_attention(a, 64, s));
    ORCCHK(gemm(e->w_att, d, L.o, L.bo, e->w_h, d, e->w_h, d, M, EPI_RESIDUAL, s, false));
    HIPCHK(launch_layernorm(e->w_h, d, L.ln2w, L.ln2b, e->w_xn, d, M, d, c.clip_eps, s));
    ORCCHK(gemm(e->w_xn, d, L.fc1, L.b1, nullptr, 0, e->w_mlp, c.clip_ff, M, EPI_QUICKGELU, s, false));
    ORCCHK(gemm(e->w_mlp, c.clip_ff, L.fc2, L.b2, e->w_h, d, e->w_h, d, M, EPI_RESIDUAL, s, false));
  }
  return 0;
}

extern "C" int orc_vision_encode(orc_engine* e, const void* images, int n_images, void* out, void* stream) {
  if (!e || !e->finalized) return fail("orc_vision_encode", "engine not finalized");
  const orc_config& c = e->c;
  ORCCHK(clip_forward(e, images, n_images, c.clip_layers - 1, S(stream)));
  const int G = c.clip_image / c.clip_patch;
  HIPCHK(launch_strip_cls(e->w_h, (bf16_t*)out, n_images, G * G + 1, c.clip_d, S(stream)));
  return 0;
}

extern "C" int orc_vision_global(orc_engine* e, const void* images, int n_images, void* out, void* stream) {
  if (!e || !e->finalized) return fail("orc_vision_global", "engine not finalized");
  const orc_config& c = e->c;
  ORCCHK(clip_forward(e, images, n_images, c.clip_layers, S(stream)));
  const int G = c.clip_image / c.clip_patch;
  // CLS rows (stride tokens*d) -> post_layernorm
  HIPCHK(launch_layernorm(e->w_h, (G * G + 1) * c.clip_d, e->post_lnw, e->post_lnb, (bf16_t*)out, c.clip_d, n_images,
                          c.clip_d, c.clip_eps, S(stream)));
  return 0;
}

extern "C" int orc_pool_views(orc_engine* e, const void* features, const int32_t* views, int B, void* out, void* stream) {
  if (!e || !e->finalized) return fail("orc_pool_views", "engine not finalized");
  const orc_config& c = e->c;
  hipStream_t s = S(stream);
  const int G = c.clip_image / c.clip_patch, patches = G * G, d = c.clip_d;
  if (B < 1 || B > c.max_batch || B > kMaxRows) return fail("orc_pool_views", "batch outside 1..min(max_batch, 32)");
  int vmax = 0, off = 0;
  ScatterArgs ro = {}, rv = {};   // per-row feature offset / valid length go to the device by value (no host staging, no sync)
  ro.n = rv.n = B; ro.dst = e->d_rowoff; rv.dst = e->d_rowvalid;
  for (int b = 0; b < B; ++b) {
    if (views[b] < 1) return fail("orc_pool_views", "a row has no views");
    ro.val[b] = off * patches;
    rv.val[b] = views[b] * patches;
    off += views[b];
    if (views[b] > vmax) vmax = views[b];
  }
  const int Sx = vmax * patches;
  if (Sx > c.pool_maxpos) return fail("orc_pool_views", "views*patches exceeds the pooler's max_position_embeddings");
  if (off > c.max_images) return fail("orc_pool_views", "too many images");
  HIPCHK(launch_scatter_ints(ro, s));
  HIPCHK(launch_scatter_ints(rv, s));
  const int M = B * Sx;
  HIPCHK(launch_bert_embed((const bf16_t*)features, e->d_rowoff, e->d_rowvalid, e->pool_tt0, e->pool_pos, nullptr, nullptr,
                           e->w_h, B, Sx, d, 0.f, s));
  HIPCHK(launch_layernorm(e->w_h, d, e->pool_elnw, e->pool_elnb, e->w_h, d, M, d, c.pool_eps, s));
  for (int i = 0; i < c.pool_layers; ++i) {
    const PoolLayer& L = e->pool[i];
    // Only the first `patches` tokens of every row leave the pooler (multimodal_projector/builder.py:80 keeps [:, :576]): in
    // the LAST layer the queries, the output projection, both LayerNorms and the MLP run on those rows only (K / V still
    // cover all Sx tokens); the reference computes the other 2/3 of that layer at 3 views and throws it away.
    const bool last = (i == c.pool_layers - 1) && Sx > patches;
    const int Sq = last ? patches : Sx, Mq = B * Sq;
    ORCCHK(gemm(e->w_h, d, L.qkv, L.bqkv, nullptr, 0, e->w_qkv, 3 * d, M, EPI_NONE, s, false));
    bf16_t* hq = e->w_h;                       // residual rows of the queries
    if (last) {
      HIPCHK(launch_copy_rows(e->w_h, (long)Sx * d, e->w_aux, (long)patches * d, B, patches, d, s));
      hq = e->w_aux;
    }
    AttnArgs a;
    a.Q = e->w_qkv; a.K = e->w_qkv + d; a.V = e->w_qkv + 2 * d;
    a.q_bs = a.k_bs = a.v_bs = (long)Sx * 3 * d; a.q_hs = a.k_hs = a.v_hs = 128; a.q_ts = a.k_ts = a.v_ts = 3 * d;
    a.O = e->w_att; a.o_bs = (long)Sq * d; a.o_hs = 128; a.o_ts = d;
    a.B = B; a.H = c.pool_heads; a.Sq = Sq; a.Sk = Sx; a.kbeg = nullptr; a.kend = e->d_rowvalid; a.causal = 0; a.q_off = 0;
    a.scale = 0.08838834764831845f;   // 128^-0.5
    HIPCHK(launch_attention(a, 128, s));
    ORCCHK(gemm(e->w_att, d, L.o, L.bo, hq, d, hq, d, Mq, EPI_RESIDUAL, s, false));
    HIPCHK(launch_layernorm(hq, d, L.ln1w, L.ln1b, hq, d, Mq, d, c.pool_eps, s));
    ORCCHK(gemm(hq, d, L.wi, L.bi, nullptr, 0, e->w_mlp, c.pool_ff, Mq, EPI_GELU, s, false));
    ORCCHK(gemm(e->w_mlp, c.pool_ff, L.wout, L.bout, hq, d, hq, d, Mq, EPI_RESIDUAL, s, false));
    HIPCHK(launch_layernorm(hq, d, L.ln2w, L.ln2b, hq, d, Mq, d, c.pool_eps, s));
    if (last) {
      HIPCHK(hipMemcpyAsync(out, hq, (size_t)Mq * d * 2, hipMemcpyDeviceToDevice, s));
      return 0;
    }
  }
  HIPCHK(launch_copy_rows(e->w_h, (long)Sx * d, (bf16_t*)out, (long)patches * d, B, patches, d, s));
  return 0;
}

extern "C" int orc_project(orc_engine* e, const void* x, int rows, void* out, void* stream) {
  if (!e || !e->finalized) return fail("orc_project", "engine not finalized");
  const orc_config& c = e->c;
  if (rows < 1 || rows > e->ws_rows) return fail("orc_project", "rows outside workspace capacity");
  ORCCHK(gemm((const bf16_t*)x, c.clip_d, e->proj0, e->proj_b0, nullptr, 0, e->w_mlp, c.d_model, rows, EPI_GELU, S(stream), false));
  ORCCHK(gemm(e->w_mlp, c.d_model, e->proj2, e->proj_b2, nullptr, 0, out, c.d_model, rows, EPI_NONE, S(stream), false));
  return 0;
}

extern "C" int orc_view_reduce(orc_engine* e, const void* x, int B, int V, int64_t n, int mode, void* out, void* stream) {
  (void)e;
  if (B < 1 || V < 1 || n < 1 || (mode != 0 && mode != 1)) return fail("orc_view_reduce", "bad argument");
  HIPCHK(launch_view_reduce((const bf16_t*)x, (bf16_t*)out, B, V, (int)n, mode, S(stream)));
  return 0;
}

extern "C" int orc_pool2x2(orc_engine* e, const void* x, int n_images, int grid, int d, void* out, void* stream) {
  (void)e;
  if (n_images < 1 || grid < 2 || (grid & 1)) return fail("orc_pool2x2", "bad argument");
  HIPCHK(launch_pool2x2((const bf16_t*)x, (bf16_t*)out, n_images, grid, d, S(stream)));
  return 0;
}

extern "C" int orc_preprocess_images(const uint8_t* rgb_hwc, int n_images, int height, int width, int out_size,
                                     const int32_t* bounds, const int32_t* coeffs, int ksize, const void* lut_bf16,
                                     const int32_t* fill_rgb_host, void* tmp, void* out, void* stream) {
  if (!rgb_hwc || !bounds || !coeffs || !lut_bf16 || !fill_rgb_host || !tmp || !out) return fail("orc_preprocess_images", "null argument");
  if (n_images < 1 || height < 1 || width < 1 || out_size < 1 || ksize < 1) return fail("orc_preprocess_images", "bad size");
  HIPCHK(launch_preprocess(rgb_hwc, n_images, height, width, out_size, bounds, coeffs, ksize, (const bf16_t*)lut_bf16,
                           fill_rgb_host[0], fill_rgb_host[1], fill_rgb_host[2], (uint8_t*)tmp, (bf16_t*)out, S(stream)));
  return 0;
}

extern "C" int orc_splice(orc_engine* e, const int32_t* codes, int rows, const void* img, const void* desc, void* out,
                          void* stream) {
  if (!e || !e->finalized) return fail("orc_splice", "engine not finalized");
  HIPCHK(launch_gather_rows(codes, e->embed, (const bf16_t*)img, (const bf16_t*)desc, (bf16_t*)out, rows, e->c.d_model, S(stream)));
  return 0;
}

// ============================================================================ LLaMA
// ssq_in: fold the RMSNorm of the input rows into this projection (W must be the matching *_dec copy); C_xf: EPI_RESIDUAL also
// writes the new hidden rows fragment-ordered
static int gemv_ex(orc_engine* e, const bf16_t* X, int ldx, const Packed& W, const bf16_t* R, void* C, int ldc, int M, int epi,
                   hipStream_t s, bf16_t* kc = nullptr, bf16_t* vc = nullptr, float* ssq_out = nullptr, int x_xf = 0, int c_xf = 0,
                   hipEvent_t ev_start = nullptr, hipEvent_t ev_stop = nullptr, const float* ssq_in = nullptr, bf16_t* C_xf = nullptr) {
  const orc_config& c = e->c;
  GemvArgs a = {};
  a.x_xf = x_xf; a.c_xf = c_xf; a.ev_start = ev_start; a.ev_stop = ev_stop;
  a.ssq_in = ssq_in; a.n_part = c.d_model / 16; a.norm_d = c.d_model; a.norm_eps = c.rms_eps; a.C_xf = C_xf;
  a.map = e->row_map;
  a.X = X; a.ldx = ldx; a.Wp = W.p; a.bias = nullptr; a.R = R; a.ldr = ldc; a.C = C; a.ldc = ldc;
  a.Wc = W.wc; a.emin = W.emin; a.patch = W.patch; a.wc_group = W.wc_group;
  a.M = M; a.N = W.N; a.K = W.K; a.Nvalid = (epi == EPI_SWIGLU) ? W.Nvalid / 2 : W.Nvalid;
  a.H = c.n_heads; a.kbeg = e->d_kbeg; a.cur_len = e->d_curlen; a.cos_tab = e->cos_tab; a.sin_tab = e->sin_tab;
  a.maxpos = e->maxpos; a.Kc = kc; a.Vc = vc; a.c_bs = e->c_bs; a.c_hs = e->c_hs;
  a.ssq_out = ssq_out;
  if (epi == EPI_ROPE_KV) { a.row_meta = e->d_rowmeta; a.row_cos = e->d_rowcos; a.row_sin = e->d_rowsin; }   // of this step (decode_one)
  hipError_t err = launch_gemv_ex(a, epi, 0, s);
  if (err != hipSuccess) return fail("launch_gemv_ex", hipGetErrorString(err));
  return 0;
}

// prefill: tiled MFMA GEMMs + flash attention over all B*T positions
// pm: batch row -> KV-cache slot the row is prefilled into. Leaves the final hidden state of the LAST position of every row in
// d_h (B rows, row-major). packed: the B prompts lie one behind the other instead (T, pos and pm are not used).
static int llama_prefill_layers(orc_engine* e, bf16_t* h, bf16_t* xn, bf16_t* qkv, bf16_t* att, bf16_t* mlp, int B, int T,
                                const int32_t* pos, hipStream_t s, const RowMap& pm, const PackedRows* packed = nullptr) {
  const orc_config& c = e->c;
  const int d = c.d_model, M = packed ? packed->start[B] : B * T;
  int n_work = 0;
  if (packed) {
    n_work = launch_attn_plan(*packed, e->d_plan, s);
    if (n_work < 0) return -1;
  }
  for (int i = 0; i < c.n_layers; ++i) {
    const LlamaLayer& L = e->llama[i];
    bf16_t* kc = e->kcache + (size_t)i * e->kv_layer_elems;
    bf16_t* vc = e->vcache + (size_t)i * e->kv_layer_elems;
    HIPCHK(launch_rmsnorm(h, d, L.ln_in, xn, d, M, d, c.rms_eps, s));
    ORCCHK(gemm(xn, d, L.qkv, nullptr, nullptr, 0, qkv, 3 * d, M, EPI_NONE, s, false));
    RopeArgs r;
    r.qkv = qkv; r.B = B; r.T = T; r.H = c.n_heads; r.pos = pos; r.kbeg = e->d_kbeg; r.cur_len = e->d_curlen;
    r.cos_tab = e->cos_tab; r.sin_tab = e->sin_tab; r.maxpos = e->maxpos; r.Kc = kc; r.Vc = vc; r.c_bs = e->c_bs; r.c_hs = e->c_hs;
    r.t0 = 0; r.map = pm;
    if (packed) {
      HIPCHK(launch_rope_packed(r, *packed, s));
      const int64_t st[8] = {3 * d, 128, 3 * d, 128, 3 * d, 128, d, 128};
      ORCCHK(orc_attention_packed(qkv, qkv + d, qkv + 2 * d, att, st, e->d_plan, n_work, M, c.n_heads, c.n_heads, 128, 0, 0.08838834764831845f, s));
    } else {
      HIPCHK(launch_rope_kv(r, s));
      AttnArgs a;
      a.Q = qkv; a.q_bs = (long)T * 3 * d; a.q_hs = 128; a.q_ts = 3 * d;
      a.K = kc; a.k_bs = e->c_bs; a.k_hs = e->c_hs; a.k_ts = 128;
      a.V = vc; a.v_bs = e->c_bs; a.v_hs = e->c_hs; a.v_ts = 128;
      a.O = att; a.o_bs = (long)T * d; a.o_hs = 128; a.o_ts = d;
      a.B = B; a.H = c.n_heads; a.Sq = T; a.Sk = T; a.kbeg = e->d_pfkbeg; a.kend = nullptr; a.causal = 1; a.q_off = 0;
      a.scale = 0.08838834764831845f;
      a.kv_map_on = 1; a.kv_map = pm;
      HIPCHK(launch_attention(a, 128, s));
    }
    if (i == c.n_layers - 1) {
      // Greedy search reads only the last position of every row (the reference computes logits for all T and discards them,
      // llava_llama.py:87-98), and nothing after the last layer's K / V write depends on the other positions: its o_proj and MLP
      // run on the B last rows only, through the decode GEMVs on the same packed weights (M = B <= 32).
      if (packed) {
        HIPCHK(launch_last_rows(att, *packed, e->d_att, d, s));
        HIPCHK(launch_last_rows(h, *packed, e->d_h, d, s));
      } else {
        HIPCHK(launch_copy_rows(att + (size_t)(T - 1) * d, (long)T * d, e->d_att, d, B, 1, d, s));
        HIPCHK(launch_copy_rows(h + (size_t)(T - 1) * d, (long)T * d, e->d_h, d, B, 1, d, s));
      }
      ORCCHK(gemm(e->d_att, d, L.o, nullptr, e->d_h, d, e->d_h, d, B, EPI_RESIDUAL, s, true));
      HIPCHK(launch_rmsnorm(e->d_h, d, L.ln_post, e->d_xn, d, B, d, c.rms_eps, s));
      ORCCHK(gemm(e->d_xn, d, L.gu, nullptr, nullptr, 0, e->d_mlp, c.d_ff, B, EPI_SWIGLU, s, true));
      ORCCHK(gemm(e->d_mlp, c.d_ff, L.down, nullptr, e->d_h, d, e->d_h, d, B, EPI_RESIDUAL, s, true));
      break;
    }
    ORCCHK(gemm(att, d, L.o, nullptr, h, d, h, d, M, EPI_RESIDUAL, s, false));
    HIPCHK(launch_rmsnorm(h, d, L.ln_post, xn, d, M, d, c.rms_eps, s));
    ORCCHK(gemm(xn, d, L.gu, nullptr, nullptr, 0, mlp, c.d_ff, M, EPI_SWIGLU, s, false));
    ORCCHK(gemm(mlp, c.d_ff, L.down, nullptr, h, d, h, d, M, EPI_RESIDUAL, s, false));
  }
  return 0;
}

// decode: 5 launches per layer; the activations between them (d_hxf, d_att, d_mlp) are kept in the fragment-ordered
// layout of common.h xf_off, written so by their producers --
//   [qkv GEMV (input RMSNorm folded in) + rotary + KV write] [attention over the cache]
//   [o_proj GEMV + residual + ssq partials] [gate/up GEMV (post-attention RMSNorm folded in) + SiLU*mul]
//   [down GEMV + residual + ssq partials]
// The residual epilogues leave per-n-tile sums of squares of the new hidden state in d_ssq and the hidden rows themselves
// fragment-ordered in d_hxf; the projection that follows reads the RAW rows, its weight copy carries the norm weight
// (W' = bf16(W * w_norm)) and its epilogue multiplies row b by rsqrt(mean(h_b^2) + eps) before the first rounding.
// Rounding points that move against the reference's eager RMSNorm -> Linear: the normalised activation is no longer
// rounded to bf16 twice (after the scale, after the weight), the folded weight is rounded once more instead.
static int llama_decode_layers(orc_engine* e, int B, hipStream_t s, bool skip_finished) {
  const orc_config& c = e->c;
  const int d = c.d_model;
  bf16_t *h = e->d_h, *hxf = e->d_hxf, *q = e->d_qkv, *att = e->d_att, *mlp = e->d_mlp;
  for (int i = 0; i < c.n_layers; ++i) {
    const LlamaLayer& L = e->llama[i];
    bf16_t* kc = e->kcache + (size_t)i * e->kv_layer_elems;
    bf16_t* vc = e->vcache + (size_t)i * e->kv_layer_elems;
    if (e->fold_norm) {
      ORCCHK(gemv_ex(e, hxf, d, L.qkv_dec, nullptr, q, d, B, EPI_ROPE_KV, s, kc, vc, nullptr, 1, 0, nullptr, nullptr, e->d_ssq));
    } else {   // ORC_DECODE_NORM=exact
      HIPCHK(launch_rmsnorm(h, d, L.ln_in, e->d_xn, d, B, d, c.rms_eps, s));
      ORCCHK(gemv_ex(e, e->d_xn, d, L.qkv_dec, nullptr, q, d, B, EPI_ROPE_KV, s, kc, vc, nullptr, 0, 0));
    }
    DecodeAttnArgs a;
    a.o_xf = 1;
    a.Q = q; a.q_bs = d; a.Kc = kc; a.Vc = vc; a.c_bs = e->c_bs; a.c_hs = e->c_hs; a.O = att; a.o_bs = d;
    a.part = e->w_part; a.kbeg = e->d_kbeg; a.cur_len = e->d_curlen; a.B = B; a.H = c.n_heads;
    a.unfinished = skip_finished ? e->d_unf : nullptr;
    a.map = e->row_map;
    a.scale = 0.08838834764831845f;
    HIPCHK(launch_decode_attention(a, s));
    ORCCHK(gemv_ex(e, att, d, L.o, h, h, d, B, EPI_RESIDUAL, s, nullptr, nullptr, e->d_ssq, 1, 0, nullptr, nullptr, nullptr, hxf));
    // sampled launches carry their own start / stop events (the dispatch's timestamps, not a pair of event commands
    // around it, which would add the launch boundary). An event-carrying launch costs the step ~6 us (measured: 596 samples per
    // generate() call = 3-4 ms, tools/generate_prof.py), so one launch is sampled every 4th token, at layer 0 / 8 / 16 / 24 in turn
    // (37 samples per 150-token call).
    const bool sample = e->prof_on && (e->steps_issued & 3) == 0 && i == ((e->steps_issued >> 2) & 3) * 8 && i < c.n_layers &&
                        e->ev_used < (int)e->ev_a.size();
    if (!e->fold_norm) HIPCHK(launch_rmsnorm(h, d, L.ln_post, e->d_xn, d, B, d, c.rms_eps, s));
    ORCCHK(gemv_ex(e, e->fold_norm ? hxf : e->d_xn, d, L.gu_dec, nullptr, mlp, c.d_ff, B, EPI_SWIGLU, s, nullptr, nullptr, nullptr, e->fold_norm ? 1 : 0, 1,
                   sample ? e->ev_a[e->ev_used] : nullptr, sample ? e->ev_b[e->ev_used] : nullptr, e->fold_norm ? e->d_ssq : nullptr));
    if (sample) ++e->ev_used;
    ORCCHK(gemv_ex(e, mlp, c.d_ff, L.down, h, h, d, B, EPI_RESIDUAL, s, nullptr, nullptr, e->d_ssq, 1, 0, nullptr, nullptr, nullptr, hxf));
  }
  return 0;
}

// final RMSNorm + lm_head + greedy sampling of B rows; row i owns the state of slot sm.slot[i].
// from_decode: hrows = d_h with fresh partials in d_ssq and the raw rows in d_hxf (the decode rows, sm = the decode map).
static int head_and_sample(orc_engine* e, const bf16_t* hrows, int ldh, int B, float* logits_out, bool from_decode, hipStream_t s,
                           const RowMap& sm, bool freeze = true) {
  const orc_config& c = e->c;
  if (from_decode && !e->fold_norm) {   // ORC_DECODE_NORM=exact
    HIPCHK(launch_rmsnorm(e->d_h, c.d_model, e->final_norm, e->d_xn, c.d_model, B, c.d_model, c.rms_eps, s));
    ORCCHK(gemv_ex(e, e->d_xn, c.d_model, e->lm_head_dec, nullptr, e->w_logits, c.vocab, B, EPI_F32, s));
  } else if (from_decode) {   // final RMSNorm folded into the lm_head projection (raw rows in d_hxf, partials in d_ssq)
    ORCCHK(gemv_ex(e, e->d_hxf, c.d_model, e->lm_head_dec, nullptr, e->w_logits, c.vocab, B, EPI_F32, s, nullptr, nullptr, nullptr, 1, 0,
                   nullptr, nullptr, e->d_ssq));
  } else {
    HIPCHK(launch_rmsnorm(hrows, ldh, e->final_norm, e->d_xn, c.d_model, B, c.d_model, c.rms_eps, s));
    ORCCHK(gemv_ex(e, e->d_xn, c.d_model, e->lm_head, nullptr, e->w_logits, c.vocab, B, EPI_F32, s));
  }
  if (logits_out)
    HIPCHK(hipMemcpyAsync(logits_out, e->w_logits, (size_t)B * c.vocab * 4, hipMemcpyDeviceToDevice, s));
  SampleArgs a;
  a.logits = e->w_logits; a.vocab = c.vocab; a.B = B; a.map = sm; a.count = e->row_map; a.n_count = e->cur_batch;
  a.unfinished = e->d_unf; a.next_ids = e->d_next;
  a.raw_argmax = e->d_argmax; a.out_tokens = e->d_tokens; a.out_ld = c.max_new_tokens; a.row_step = e->d_rowstep;
  a.cur_len = e->d_curlen; a.limit = e->d_limit; a.step = e->d_step; a.n_unfinished = e->d_nunf;
  a.pad_id = c.pad_token_id; a.eos_id = c.eos_token_id; a.freeze_finished = freeze ? 1 : 0;
  HIPCHK(launch_argmax_sample(a, s));
  return 0;
}

// LlavaLlamaForCausalLM.forward step 0 for k left-padded rows into the KV-cache slots slots[0..k): resets those slots'
// greedy state (one small launch, no host staging), runs the 32 layers over all k * T positions, samples each row's first token.
// lens: the rows' prompts lie one behind the other without padding instead, lens[i] rows each (position_ids, left_pad and T are not used).
static int prefill_into_slots(orc_engine* e, const int* slots, int k, const void* embeds, const int32_t* position_ids,
                              const int32_t* left_pad, const int32_t* limits, int T, float* logits_out, hipStream_t s, const char* who,
                              const int32_t* lens = nullptr) {
  const orc_config& c = e->c;
  if (k < 1 || k > c.max_batch || k > kMaxRows) return fail(who, "row count outside 1..min(max_batch, 32)");
  PackedRows pr = {};
  if (lens) {
    for (int i = 0; i < k; ++i) {
      if (lens[i] < 1 || lens[i] >= c.max_seq) return fail(who, "prompt length outside 1..max_seq-1");
      pr.start[i + 1] = pr.start[i] + lens[i];   // at most 32 x max_seq
    }
    pr.n = k;
  } else if (T < 1 || T >= c.max_seq) {
    return fail(who, "prompt length exceeds max_seq");
  }
  if ((lens ? (long)pr.start[k] : (long)k * T) > e->ws_rows) return fail(who, "rows*T exceeds workspace");
  SlotInitArgs in = {};
  RowMap pm;
  for (int i = 0; i < kMaxRows; ++i) pm.slot[i] = -1;
  for (int i = 0; i < k; ++i) {
    if (slots[i] < 0 || slots[i] >= c.max_batch) return fail(who, "slot outside 0..max_batch-1");
    for (int j = 0; j < i; ++j)
      if (slots[j] == slots[i]) return fail(who, "a slot is named twice");
    if (lens) T = lens[i];
    if (!lens && (left_pad[i] < 0 || left_pad[i] >= T)) return fail(who, "left_pad outside 0..T-1");
    const int lim = limits ? limits[i] : c.max_new_tokens;
    if (lim < 1 || lim > c.max_new_tokens) return fail(who, "length stop outside 1..max_new_tokens");
    if (limits && T + lim > c.max_seq) return fail(who, "prompt + length stop exceeds max_seq");
    pm.slot[i] = slots[i];
    in.kbeg[i] = lens ? 0 : left_pad[i];
    in.limit[i] = lim;
    in.T[i] = T;
  }
  pr.map = pm;
  in.map = pm; in.k = k; in.pad_id = c.pad_token_id; in.out_ld = c.max_new_tokens;
  in.unfinished = e->d_unf; in.kbeg_state = e->d_kbeg; in.cur_len = e->d_curlen; in.row_step = e->d_rowstep; in.limit_state = e->d_limit;
  in.tokens = e->d_tokens; in.pf_kbeg = e->d_pfkbeg;
  HIPCHK(launch_slot_init(in, s));
  const int d = c.d_model, M = lens ? pr.start[k] : k * T;
  HIPCHK(hipMemcpyAsync(e->w_h, embeds, (size_t)M * d * 2, hipMemcpyDeviceToDevice, s));
  ORCCHK(llama_prefill_layers(e, e->w_h, e->w_xn, e->w_qkv, e->w_att, e->w_mlp, k, T, position_ids, s, pm, lens ? &pr : nullptr));
  ORCCHK(head_and_sample(e, e->d_h, d, k, logits_out, false, s, pm));   // the rows' last positions
  return 0;
}

extern "C" int orc_prefill(orc_engine* e, const void* embeds, const int32_t* position_ids, const int32_t* left_pad,
                           int B, int T, float* logits_out, void* stream) {
  if (!e || !e->finalized) return fail("orc_prefill", "engine not finalized");
  hipStream_t s = S(stream);
  if (B < 1 || B > e->c.max_batch || B > kMaxRows) return fail("orc_prefill", "batch outside 1..min(max_batch, 32)");
  int slots[kMaxRows];
  for (int i = 0; i < kMaxRows; ++i) {
    slots[i] = i;
    e->row_map.slot[i] = i < B ? i : -1;   // decode row b <-> slot b
  }
  e->stream_mode = false;
  e->cur_batch = B;
  e->cur_T = T;
  e->steps_issued = 0;
  HIPCHK(hipMemsetAsync(e->dev_ints, 0, 16 * 4, s));   // step = 0; n_unfinished is set by the sampler
  return prefill_into_slots(e, slots, B, embeds, position_ids, left_pad, nullptr, T, logits_out, s, "orc_prefill");
}

// decode step k (1-based since the prefill) writes K/V slot T + k - 1 of every row: refuse the step that would leave the
// cache (the device counters are only mirrored here; nothing on the device bounds the slot)
static int check_capacity(orc_engine* e, int n_steps, const char* who) {
  if (n_steps < 0) return fail(who, "negative step count");
  if (e->stream_mode) return 0;   // every slot was admitted with T + length stop <= max_seq and freezes at its stop
  if (e->cur_T + e->steps_issued + n_steps > e->c.max_seq) {
    char msg[160];
    snprintf(msg, sizeof(msg), "KV cache full: prompt %d + %d steps taken + %d requested > max_seq %d", e->cur_T, e->steps_issued,
             n_steps, e->c.max_seq);
    return fail(who, msg);
  }
  return 0;
}

static int decode_one(orc_engine* e, const int32_t* forced, float* logits_out, hipStream_t s) {
  const orc_config& c = e->c;
  const int B = e->cur_batch;
  ++e->steps_issued;
  RowMetaArgs rm;
  rm.cur_len = e->d_curlen; rm.kbeg = e->d_kbeg; rm.unfinished = e->d_unf; rm.cos_tab = e->cos_tab; rm.sin_tab = e->sin_tab;
  rm.maxpos = e->maxpos; rm.row_meta = e->d_rowmeta; rm.row_cos = e->d_rowcos; rm.row_sin = e->d_rowsin;
  HIPCHK(launch_embed_tokens(forced, e->d_next, e->row_map, e->embed, e->d_h, B, c.d_model, c.vocab, e->d_ssq, c.d_model / 16, s, e->d_hxf, &rm));
  // free-running: finished rows freeze (their tokens are pad, their cache is not read or grown); teacher forcing: every
  // row advances with the forced token whatever the sampler thinks
  ORCCHK(llama_decode_layers(e, B, s, forced == nullptr));
  ORCCHK(head_and_sample(e, e->d_h, c.d_model, B, logits_out, true, s, e->row_map, forced == nullptr));
  return 0;
}

extern "C" int orc_decode_step(orc_engine* e, const int32_t* forced_ids, float* logits_out, void* stream) {
  if (!e || !e->finalized || e->cur_batch == 0) return fail("orc_decode_step", "no prefill has run");
  if (e->stream_mode && forced_ids) return fail("orc_decode_step", "teacher forcing is not available between orc_stream_begin and the next orc_prefill");
  ORCCHK(check_capacity(e, 1, "orc_decode_step"));
  return decode_one(e, forced_ids, logits_out, S(stream));
}

extern "C" int orc_decode_steps(orc_engine* e, int n_steps, void* stream) {
  if (!e || !e->finalized || e->cur_batch == 0) return fail("orc_decode_steps", "no prefill has run");
  ORCCHK(check_capacity(e, n_steps, "orc_decode_steps"));
  for (int i = 0; i < n_steps; ++i) ORCCHK(decode_one(e, nullptr, nullptr, S(stream)));
  return 0;
}

extern "C" int orc_read_state(orc_engine* e, int32_t* tokens_host, int32_t* steps_host, int32_t* n_unf_host,
                              int32_t* last_argmax_host, void* stream) {
  if (!e || !e->finalized) return fail("orc_read_state", "engine not finalized");
  if (e->stream_mode) return fail("orc_read_state", "use orc_read_slots between orc_stream_begin and the next orc_prefill");
  hipStream_t s = S(stream);
  int hdr[16];
  HIPCHK(hipMemcpyAsync(hdr, e->dev_ints, 16 * 4, hipMemcpyDeviceToHost, s));
  if (tokens_host && e->cur_batch > 0)
    HIPCHK(hipMemcpyAsync(tokens_host, e->d_tokens, (size_t)e->cur_batch * e->c.max_new_tokens * 4, hipMemcpyDeviceToHost, s));
  if (last_argmax_host && e->cur_batch > 0)
    HIPCHK(hipMemcpyAsync(last_argmax_host, e->d_argmax, (size_t)e->cur_batch * 4, hipMemcpyDeviceToHost, s));
  HIPCHK(hipStreamSynchronize(s));
  if (steps_host) *steps_host = hdr[0];
  if (n_unf_host) *n_unf_host = hdr[2];
  return 0;
}

extern "C" int orc_set_row_limits(orc_engine* e, const int32_t* limits_host, int n, void* stream) {
  if (!e || !e->finalized || e->cur_batch == 0) return fail("orc_set_row_limits", "no prefill has run");
  if (!limits_host || n != e->cur_batch) return fail("orc_set_row_limits", "one limit per row of the running batch");
  ScatterArgs sa = {};
  sa.map = e->row_map; sa.n = n; sa.dst = e->d_limit;
  for (int i = 0; i < n; ++i) {
    if (limits_host[i] < 1 || limits_host[i] > e->c.max_new_tokens) return fail("orc_set_row_limits", "limit outside 1..max_new_tokens");
    sa.val[i] = limits_host[i];
  }
  HIPCHK(launch_scatter_ints(sa, S(stream)));
  // limit 1: the prefill has already sampled the row's only token (under the default limit, so its flag may still say
  // "unfinished"): mark those rows finished now, or the first decode step would emit a second token for them.
  // Rows are only ever moved to "finished" here, so a row that ended on EOS stays finished.
  ScatterArgs fin = {};
  fin.n = n; fin.dst = e->d_unf;
  bool any = false;
  for (int i = 0; i < kMaxRows; ++i) fin.map.slot[i] = -1;
  for (int i = 0; i < n; ++i)
    if (limits_host[i] == 1) { fin.map.slot[i] = e->row_map.slot[i]; fin.val[i] = 0; any = true; }
  if (any) HIPCHK(launch_scatter_ints(fin, S(stream)));
  return 0;
}

// ---------------------------------------------------------------------------- continuous batching
extern "C" int orc_stream_begin(orc_engine* e, int n_rows, void* stream) {
  if (!e || !e->finalized) return fail("orc_stream_begin", "engine not finalized");
  if (n_rows < 1 || n_rows > e->c.max_batch || n_rows > kMaxRows) return fail("orc_stream_begin", "n_rows outside 1..min(max_batch, 32)");
  hipStream_t s = S(stream);
  e->stream_mode = true;
  e->cur_batch = n_rows;
  e->cur_T = 0;
  e->steps_issued = 0;
  for (int i = 0; i < kMaxRows; ++i) e->row_map.slot[i] = -1;   // no decode row is attached to a slot yet
  HIPCHK(hipMemsetAsync(e->dev_ints, 0, DI_TOKENS * 4, s));
  return 0;
}

extern "C" int orc_prefill_slots(orc_engine* e, const int32_t* slots_host, int n, const void* embeds, const int32_t* position_ids,
                                 const int32_t* left_pad_host, const int32_t* limits_host, int T, float* logits_out, void* stream) {
  if (!e || !e->finalized) return fail("orc_prefill_slots", "engine not finalized");
  if (!e->stream_mode) return fail("orc_prefill_slots", "call orc_stream_begin first");
  if (!slots_host || !embeds || !position_ids || !left_pad_host || !limits_host) return fail("orc_prefill_slots", "null argument");
  for (int i = 0; i < n && i < kMaxRows; ++i)
    for (int r = 0; r < e->cur_batch; ++r)
      if (e->row_map.slot[r] == slots_host[i]) return fail("orc_prefill_slots", "slot is attached to a decode row");
  return prefill_into_slots(e, slots_host, n, embeds, position_ids, left_pad_host, limits_host, T, logits_out, S(stream), "orc_prefill_slots");
}

extern "C" int orc_prefill_packed(orc_engine* e, const int32_t* slots_host, int n, const void* embeds, const int32_t* lens_host,
                                  const int32_t* limits_host, float* logits_out, void* stream) {
  const char* who = "orc_prefill_packed";
  if (!e || !e->finalized) return fail(who, "engine not finalized");
  if (!e->stream_mode) return fail(who, "call orc_stream_begin first");
  if (!slots_host || !embeds || !lens_host || !limits_host) return fail(who, "null argument");
  for (int i = 0; i < n && i < kMaxRows; ++i)
    for (int r = 0; r < e->cur_batch; ++r)
      if (e->row_map.slot[r] == slots_host[i]) return fail(who, "slot is attached to a decode row");
  return prefill_into_slots(e, slots_host, n, embeds, nullptr, nullptr, limits_host, 0, logits_out, S(stream), who, lens_host);
}

extern "C" int orc_stream_attach(orc_engine* e, int row, int slot) {
  if (!e || !e->finalized || !e->stream_mode) return fail("orc_stream_attach", "call orc_stream_begin first");
  if (row < 0 || row >= e->cur_batch) return fail("orc_stream_attach", "row outside the decode width");
  if (slot < -1 || slot >= e->c.max_batch) return fail("orc_stream_attach", "slot outside -1..max_batch-1");
  for (int r = 0; r < e->cur_batch; ++r)
    if (slot >= 0 && r != row && e->row_map.slot[r] == slot) return fail("orc_stream_attach", "slot is attached to another row");
  e->row_map.slot[row] = slot;
  return 0;
}

extern "C" int orc_read_slots(orc_engine* e, int32_t* tokens_host, int32_t* row_steps_host, int32_t* unfinished_host,
                              void* stream) {
  if (!e || !e->finalized) return fail("orc_read_slots", "engine not finalized");
  hipStream_t s = S(stream);
  const int B = e->c.max_batch;
  if (tokens_host) HIPCHK(hipMemcpyAsync(tokens_host, e->d_tokens, (size_t)B * e->c.max_new_tokens * 4, hipMemcpyDeviceToHost, s));
  if (row_steps_host) HIPCHK(hipMemcpyAsync(row_steps_host, e->d_rowstep, (size_t)B * 4, hipMemcpyDeviceToHost, s));
  if (unfinished_host) HIPCHK(hipMemcpyAsync(unfinished_host, e->d_unf, (size_t)B * 4, hipMemcpyDeviceToHost, s));
  HIPCHK(hipStreamSynchronize(s));
  return 0;
}

extern "C" int orc_profile_enable(orc_engine* e, int on) {
  if (!e) return fail("orc_profile_enable", "null engine");
  if (on && e->ev_a.empty()) {
    e->ev_a.resize(4096);
    e->ev_b.resize(4096);
    for (size_t i = 0; i < e->ev_a.size(); ++i) {
      HIPCHK(hipEventCreate(&e->ev_a[i]));
      HIPCHK(hipEventCreate(&e->ev_b[i]));
    }
  }
  e->prof_on = on != 0;
  e->ev_used = 0;
  return 0;
}

extern "C" int orc_profile_read(orc_engine* e, double* total_ms, int32_t* count, int64_t* bytes_per_launch) {
  if (!e) return fail("orc_profile_read", "null engine");
  HIPCHK(hipDeviceSynchronize());
  double tot = 0.0;
  for (int i = 0; i < e->ev_used; ++i) {
    float ms = 0.f;
    HIPCHK(hipEventElapsedTime(&ms, e->ev_a[i], e->ev_b[i]));
    tot += ms;
  }
  if (total_ms) *total_ms = tot;
  if (count) *count = e->ev_used;
  // algorithmic bytes of one gate/up GEMV launch: the two weight matrices (activations are L2-resident and small)
  if (bytes_per_launch) *bytes_per_launch = (int64_t)2 * 2 * e->c.d_ff * e->c.d_model;
  return 0;
}

extern "C" int64_t orc_decode_weight_bytes(orc_engine* e) {
  const orc_config& c = e->c;
  const int64_t per_layer = (int64_t)4 * c.d_model * c.d_model + (int64_t)3 * c.d_model * c.d_ff + 2 * c.d_model;
  return 2 * (per_layer * c.n_layers + c.d_model + (int64_t)c.vocab * c.d_model);
}
static int64_t stream_bytes(const Packed& W) {
  const int64_t nk = (int64_t)W.N * W.K;
  return W.wc ? nk * 3 / 2 + nk / 512 : nk * 2;
}
extern "C" int64_t orc_decode_stream_bytes(orc_engine* e, int which) {
  if (!e || !e->finalized || e->llama.empty()) return 0;
  if (which == 1) return stream_bytes(e->llama[0].gu_dec);
  int64_t t = stream_bytes(e->lm_head_dec) + (int64_t)2 * e->c.d_model;
  for (const LlamaLayer& L : e->llama) t += stream_bytes(L.qkv_dec) + stream_bytes(L.o) + stream_bytes(L.gu_dec) + stream_bytes(L.down);
  return t;
}
extern "C" int orc_decode_weight_stats(orc_engine* e, int64_t* out6) {
  if (!e || !e->finalized || !out6) return fail("orc_decode_weight_stats", "engine not finalized / null output");
  out6[0] = e->cw_mats; out6[1] = e->cw_done; out6[2] = e->cw_elems; out6[3] = e->cw_escapes;
  out6[4] = e->cw_blocks; out6[5] = e->cw_flagged_blocks;
  return 0;
}
extern "C" int64_t orc_kv_bytes_per_key(orc_engine* e) { return (int64_t)2 * 2 * e->c.n_layers * e->c.d_model; }

// ============================================================================ single-kernel hooks
extern "C" int orc_test_gemm(const void* x, int M, int K, const void* w, int N, const void* bias, const void* residual,
                             int epi, int use_gemv, void* out, void* stream) {
  hipStream_t s = S(stream);
  const int Np = round_up(N, 256), Kp = round_up(K, 64);
  if (Kp != K) return fail("orc_test_gemm", "K must be a multiple of 64");
  bf16_t* wp;
  HIPCHK(hipMalloc((void**)&wp, (size_t)Np * Kp * 2));
  int* rm = nullptr;
  if (epi == EPI_SWIGLU) {   // w = [gate(N/2 rows); up(N/2 rows)] -> interleave 16-row tiles
    std::vector<int> m(Np, -1);
    for (int pr = 0; pr < N; ++pr) {
      const int t = pr / 32, wi = pr % 32;
      m[pr] = wi < 16 ? 16 * t + wi : N / 2 + 16 * t + (wi - 16);
    }
    HIPCHK(hipMalloc((void**)&rm, Np * 4));
    HIPCHK(hipMemcpy(rm, m.data(), Np * 4, hipMemcpyHostToDevice));
  }
  HIPCHK(launch_pack_weight((const bf16_t*)w, N, K, rm, wp, Np, Kp, s));
  GemmArgs a;
  a.X = (const bf16_t*)x; a.ldx = K; a.Wp = wp; a.bias = (const bf16_t*)bias; a.R = (const bf16_t*)residual;
  const int nout = epi == EPI_SWIGLU ? N / 2 : N;
  a.ldr = nout; a.C = out; a.ldc = nout; a.M = M; a.N = Np; a.K = Kp; a.Nvalid = nout;
  // use_gemv: 0 = GEMM (automatic kernel choice), 1 = decode GEMV, 2 = 128^2 register-staged GEMM, 3 / 4 = LDS-DMA GEMM with
  // 256-row / 128-row tiles only, 5 = decode GEMV on the lossless 12-bit copy of the weights (must equal 1 bit for bit),
  // 6 / 7 = 1 / 5 on the r2 kernels (branchy k-loop; must equal the pipelined kernels bit for bit), 8 = 5 with row-major compressed blocks,
  // 100 + n = LDS-DMA GEMM with n 256-row m-tiles and 128-row tiles for the remaining rows
  hipError_t err;
  struct LegacyGuard { ~LegacyGuard() { gemv_force_legacy(0); } } legacy_guard;
  if (use_gemv == 6 || use_gemv == 7) {
    gemv_force_legacy(1);
    use_gemv = use_gemv == 6 ? 1 : 5;
  }
  const int test_group = use_gemv == 8 ? 0 : kCwGroup;   // 8 = 5 with the compressed blocks in row-major order (must equal 5 bit for bit)
  if (use_gemv == 8) use_gemv = 5;
  if (use_gemv == 5) {
    const int nt_unit = gemv_unit_tiles(epi, Np), units = Np / 16 / nt_unit;
    const size_t nblk = (size_t)(Np / 16) * (Kp / 32);
    uint8_t *wc, *em;
    uint16_t* patch;
    int* cnt;
    HIPCHK(hipMalloc((void**)&wc, nblk * 768));
    HIPCHK(hipMalloc((void**)&em, (nblk + 7) & ~(size_t)3));
    HIPCHK(hipMalloc((void**)&patch, (size_t)units * 256 * 2));
    HIPCHK(hipMalloc((void**)&cnt, (size_t)(units + 1) * 4));
    HIPCHK(hipMemsetAsync(cnt + units, 0, 4, s));
    HIPCHK(launch_compress_weight(wp, Np, Kp, nt_unit, wc, em, patch, cnt, cnt + units, s, test_group));
    int overflow = 0;
    HIPCHK(hipMemcpyAsync(&overflow, cnt + units, 4, hipMemcpyDeviceToHost, s));
    HIPCHK(hipStreamSynchronize(s));
    err = hipSuccess;
    if (!overflow) {
      GemvArgs g = {};
      g.map = identity_map();
      g.X = a.X; g.ldx = a.ldx; g.Wp = nullptr; g.Wc = wc; g.emin = em; g.patch = patch; g.wc_group = test_group; g.bias = a.bias; g.R = a.R; g.ldr = a.ldr;
      g.C = a.C; g.ldc = a.ldc; g.M = a.M; g.N = a.N; g.K = a.K; g.Nvalid = a.Nvalid;
      err = launch_gemv_ex(g, epi, 0, s);
      HIPCHK(hipStreamSynchronize(s));
    }
    HIPCHK(hipFree(wc)); HIPCHK(hipFree(em)); HIPCHK(hipFree(patch)); HIPCHK(hipFree(cnt));
    HIPCHK(hipFree(wp));
    if (rm) HIPCHK(hipFree(rm));
    if (overflow) return fail("orc_test_gemm", "weights not compressible: a unit has more than 254 non-zero out-of-range elements");
    if (err != hipSuccess) return fail("orc_test_gemm", hipGetErrorString(err));
    return 0;
  }
  if (use_gemv >= 100) gemm_force_kernel(use_gemv);
  else if (use_gemv >= 2) gemm_force_kernel(use_gemv - 1);
  err = use_gemv == 1 ? launch_gemv(a, epi, s) : launch_gemm(a, epi, s);
  gemm_force_kernel(0);
  if (err != hipSuccess) return fail("orc_test_gemm", hipGetErrorString(err));
  HIPCHK(hipStreamSynchronize(s));
  HIPCHK(hipFree(wp));
  if (rm) HIPCHK(hipFree(rm));
  return 0;
}

// RMSNorm -> Linear at decode shapes, both ways (tests/test_kernels_gpu.py::test_folded_rmsnorm_against_exact):
//   out_exact  = GEMV(W, rmsnorm(x; w_norm))                       the reference's rounding points (the prefill's norm kernel)
//   out_folded = r_b * GEMV(bf16(W * diag(w_norm)), x raw)         the decode path: norm weight folded into the weight copy, row
//                                                                  scale from per-16-column partial sums of squares in the epilogue
// x (M, K) bf16, w_norm (K) bf16, w (N, K) bf16 row-major, outputs (M, N) bf16. M <= 32, K % 256 == 0, N % 256 == 0.
extern "C" int orc_test_folded_norm(const void* x, int M, int K, const void* w_norm, const void* w, int N, float eps,
                                    void* out_exact, void* out_folded, void* stream) {
  hipStream_t s = S(stream);
  if (M < 1 || M > kMaxRows || (K % 256) || (N % 256)) return fail("orc_test_folded_norm", "M in 1..32, K and N multiples of 256");
  bf16_t *wp, *wf, *xn, *xf;
  float* ssq;
  HIPCHK(hipMalloc((void**)&wp, (size_t)N * K * 2));
  HIPCHK(hipMalloc((void**)&wf, (size_t)N * K * 2));
  HIPCHK(hipMalloc((void**)&xn, (size_t)kMaxRows * K * 2));
  HIPCHK(hipMalloc((void**)&xf, (size_t)kMaxRows * K * 2));
  HIPCHK(hipMalloc((void**)&ssq, (size_t)kMaxRows * (K / 16) * 4));
  HIPCHK(launch_pack_weight((const bf16_t*)w, N, K, nullptr, wp, N, K, s));
  HIPCHK(launch_pack_weight((const bf16_t*)w, N, K, nullptr, wf, N, K, s, (const bf16_t*)w_norm));
  // the raw rows fragment-ordered + their per-16-column sums of squares, as the residual epilogues leave them: an identity
  // "token gather" over x (vocab = M, ids = row index)
  std::vector<int> ids(M);
  for (int i = 0; i < M; ++i) ids[i] = i;
  int* dids;
  HIPCHK(hipMalloc((void**)&dids, M * 4));
  HIPCHK(hipMemcpyAsync(dids, ids.data(), M * 4, hipMemcpyHostToDevice, s));
  HIPCHK(launch_embed_tokens(dids, nullptr, identity_map(), (const bf16_t*)x, xn, M, K, M, ssq, K / 16, s, xf));
  // exact
  HIPCHK(launch_rmsnorm((const bf16_t*)x, K, (const bf16_t*)w_norm, xn, K, M, K, eps, s));
  GemvArgs a = {};
  a.map = identity_map();
  a.X = xn; a.ldx = K; a.Wp = wp; a.C = out_exact; a.ldc = N; a.M = M; a.N = N; a.K = K; a.Nvalid = N;
  hipError_t err = launch_gemv_ex(a, EPI_NONE, 0, s);
  // folded
  GemvArgs f = a;
  f.X = xf; f.x_xf = 1; f.Wp = wf; f.C = out_folded; f.ssq_in = ssq; f.n_part = K / 16; f.norm_d = K; f.norm_eps = eps;
  hipError_t err2 = launch_gemv_ex(f, EPI_NONE, 0, s);
  HIPCHK(hipStreamSynchronize(s));
  HIPCHK(hipFree(wp)); HIPCHK(hipFree(wf)); HIPCHK(hipFree(xn)); HIPCHK(hipFree(xf)); HIPCHK(hipFree(ssq)); HIPCHK(hipFree(dids));
  if (err != hipSuccess || err2 != hipSuccess) return fail("orc_test_folded_norm", hipGetErrorString(err != hipSuccess ? err : err2));
  return 0;
}

extern "C" int orc_test_rmsnorm(const void* x, const void* w, int rows, int d, float eps, void* out, void* stream) {
  HIPCHK(launch_rmsnorm((const bf16_t*)x, d, (const bf16_t*)w, (bf16_t*)out, d, rows, d, eps, S(stream)));
  return 0;
}
extern "C" int orc_test_layernorm(const void* x, const void* w, const void* b, int rows, int d, float eps, void* out,
                                  void* stream) {
  HIPCHK(launch_layernorm((const bf16_t*)x, d, (const bf16_t*)w, (const bf16_t*)b, (bf16_t*)out, d, rows, d, eps, S(stream)));
  return 0;
}
// q,k,v,out contiguous (B, H, S, head_dim)
extern "C" int orc_test_attention(const void* q, const void* k, const void* v, int B, int H, int Sq, int Sk, int hd,
                                  const int32_t* kbeg, const int32_t* kend, int causal, int q_off, float scale, void* out,
                                  void* stream) {
  AttnArgs a;
  a.Q = (const bf16_t*)q; a.q_bs = (long)H * Sq * hd; a.q_hs = (long)Sq * hd; a.q_ts = hd;
  a.K = (const bf16_t*)k; a.k_bs = (long)H * Sk * hd; a.k_hs = (long)Sk * hd; a.k_ts = hd;
  a.V = (const bf16_t*)v; a.v_bs = a.k_bs; a.v_hs = a.k_hs; a.v_ts = hd;
  a.O = (bf16_t*)out; a.o_bs = a.q_bs; a.o_hs = a.q_hs; a.o_ts = hd;
  a.B = B; a.H = H; a.Sq = Sq; a.Sk = Sk; a.kbeg = kbeg; a.kend = kend; a.causal = causal; a.q_off = q_off; a.scale = scale;
  HIPCHK(launch_attention(a, hd, S(stream)));
  return 0;
}

// q (B, H*128); kcache / vcache (B, H, Tmax, 128); kbeg device (B) or null; keys [kbeg[b], n_keys) are attended.
// Runs the engine's own launch (launch_decode_attention: un-split for B*H >= 192, split + combine below). Synchronous.
extern "C" int orc_test_decode_attention(const void* q, const void* kcache, const void* vcache, int B, int H, int Tmax,
                                         const int32_t* kbeg, int n_keys, void* out, void* stream) {
  if (!q || !kcache || !vcache || !out) return fail("orc_test_decode_attention", "null argument");
  if (B < 1 || B > kMaxRows || H < 1 || Tmax < 1 || n_keys < 1 || n_keys > Tmax) return fail("orc_test_decode_attention", "bad size");
  hipStream_t s = S(stream);
  float* part = nullptr;
  int* ints = nullptr;
  HIPCHK(hipMalloc((void**)&part, (size_t)B * H * DECODE_NSPLIT * 130 * 4));
  HIPCHK(hipMalloc((void**)&ints, 64 * 4));
  int host[64] = {0};
  for (int b = 0; b < 32; ++b) host[b] = n_keys;
  HIPCHK(hipMemcpyAsync(ints, host, sizeof(host), hipMemcpyHostToDevice, s));
  if (kbeg) HIPCHK(hipMemcpyAsync(ints + 32, kbeg, B * 4, hipMemcpyDeviceToDevice, s));
  DecodeAttnArgs a;
  a.o_xf = 0;
  a.unfinished = nullptr;
  a.map = identity_map();
  a.Q = (const bf16_t*)q; a.q_bs = (long)H * 128; a.Kc = (const bf16_t*)kcache; a.Vc = (const bf16_t*)vcache;
  a.c_hs = (long)Tmax * 128; a.c_bs = a.c_hs * H; a.O = (bf16_t*)out; a.o_bs = (long)H * 128;
  a.part = part; a.kbeg = ints + 32; a.cur_len = ints; a.B = B; a.H = H; a.scale = 0.08838834764831845f;
  hipError_t err = launch_decode_attention(a, s);
  hipError_t err2 = hipStreamSynchronize(s);
  (void)hipFree(part);
  (void)hipFree(ints);
  if (err != hipSuccess) return fail("orc_test_decode_attention", hipGetErrorString(err));
  if (err2 != hipSuccess) return fail("orc_test_decode_attention", hipGetErrorString(err2));
  return 0;
}
