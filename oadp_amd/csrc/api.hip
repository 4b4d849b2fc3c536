// api.hip — the extern "C" surface of liboake_hip.so (include/oake_hip.h): handle lifetime, weight
// upload in the OpenAI-CLIP state_dict layout, the encode_image / objects-mode schedules, and the
// per-kernel HIP-event profiler that bench.py's `roofline` object reads.
//
// Schedules (reference call sites cited in include/oake_hip.h):
//   encode_image : im2col -> conv1 GEMM(+pos) -> cls+ln_pre -> 12 x { ln_1 -> QKV GEMM -> attention
//                  -> out_proj GEMM(+residual) -> ln_2 -> c_fc GEMM(+QuickGELU) -> c_proj
//                  GEMM(+residual) } -> ln_post/proj/L2-normalise head
//   objects mode : same patch/token pipeline at stride 16 (197 tokens) plus the reference Hooks'
//                  object-token stream y; the two exact savings of SURVEY.md Appendix C are taken:
//                  patch-row K/V are projected once per layer and shared by both streams, and the
//                  last layer's main stream (never read) is not executed.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <thread>
#include <atomic>
#include <vector>

#ifndef OAKE_LAB
#define OAKE_LAB 0  // 1: liboake_hip_lab.so (production kernels + the experiments that lost their A/B)
#endif
#include "../../include/oake_hip.h"
#include "../../include/oake_hip_debug.h"
#ifndef OAKE_FUSE_QKV_ATTN_DEFAULT
#define OAKE_FUSE_QKV_ATTN_DEFAULT 1  // (+2.2 % globals with two lanes, profiles/r05/ab_fuse_qkv_attn_*.log; docs/history/round5.md)
#endif
#include "kernels.h"

namespace oake {
thread_local hipEvent_t g_launch_start = nullptr, g_launch_stop = nullptr;  // common.h, OAKE_LAUNCH
}

using namespace oake;

namespace {
// Kernel-selection switches of the handle-less oake_debug_* kernel entry points (tests, tools): per
// calling thread.  Handles carry their own (oake_set_option) and never read these.
thread_local LaunchOpts t_debug_opts;


thread_local std::string g_create_error;

struct LayerW {
  float *ln1_g = nullptr, *ln1_b = nullptr, *ln2_g = nullptr, *ln2_b = nullptr;
  void *in_w = nullptr, *out_w = nullptr, *fc_w = nullptr, *proj_w = nullptr;  // 16-bit [N,K]
  float *in_b = nullptr, *out_b = nullptr, *fc_b = nullptr, *proj_b = nullptr;
  // LayerNorm folded into the consuming GEMM (16-bit residual stream; rowops.hip fold_ln_kernel):
  // fp32 masters of the two weights that follow a LayerNorm, their gamma-scaled 16-bit copies, the
  // column sums of those and the beta-shifted biases
  float *in_w32 = nullptr, *fc_w32 = nullptr;
  void *in_wf = nullptr, *fc_wf = nullptr;
  float *in_cs = nullptr, *fc_cs = nullptr, *in_bf = nullptr, *fc_bf = nullptr;
  void* out_wp = nullptr;  // out_proj weight in attn_out_kernel's fragment order (attn_out.hip), or nullptr
  // the folded in-projection in head-major row order (q | k | v per head) for qkv_attn_kernel, or nullptr
  void* in_wfp = nullptr;
  float *in_csp = nullptr, *in_bfp = nullptr;
};

struct ProfSlot {
  std::string name;
  double flops = 0, bytes = 0;
  int64_t launches = 0;  // stamped launches (what ms / flops / bytes cover)
  int64_t seen = 0;      // all launches since the reset
  double ms = 0;
};

struct PendingEvt {
  int slot;
  hipEvent_t a, b;
};

}  // namespace

struct oake_handle {
  oake_config cfg{};
  int device = 0;
  int grid = 0, tokens = 0, p2 = 0, kpatch = 0;
  int cur_len = 0;            // tokens per sequence of the pass in flight (text: <= tokens)
  int pass_cap = 0;           // crops per pass the workspace was sized for (cfg.max_batch may be lowered: OAKE_OPT_PASS_CROPS)
  bool text = false;          // text tower (oake_text_create): causal attention, token embedding
  int vocab = 0;
  float* tok_emb = nullptr;   // [vocab, width] fp32 (text)
  int dt16 = DT_F16;
  int xdt = DT_F32;           // residual-stream element type: DT_F32 or dt16
  std::string err;
  // oake_set_option: this handle's kernel-selection switches (nothing process-wide)
  LaunchOpts opts;
  int cls_last = 1;           // encode_image: last block for the CLS rows only (0 = all rows, as the reference)
  int patch_direct = 1;       // conv1 reads 16-bit NCHW input directly (0 = always through im2col; A/B, tests)
  int fuse_attn_out = 0;      // L <= 64: attention + out_proj + residual in one kernel (csrc/attn_out.hip; measured
                              // slower than the two launches — 39 vs 36 us per layer — so opt-in: tests, A/B runs)
  int fuse_qkv_attn = OAKE_FUSE_QKV_ATTN_DEFAULT;  // L <= 53: ln_1 + in_proj + attention in one kernel (csrc/qkv_attn.hip)
  bool qkv_perm = false;      // LayerW::in_wfp / in_csp / in_bfp are current

  // weights
  void* conv_w = nullptr;     // [width, 3*P*P] 16-bit
  float* cls = nullptr;       // [width]
  float* pos = nullptr;       // [tokens, width]
  float *lnpre_g = nullptr, *lnpre_b = nullptr, *lnpost_g = nullptr, *lnpost_b = nullptr;
  void* proj = nullptr;       // [embed, width] 16-bit (visual.proj transposed: GEMM W operand)
  std::vector<LayerW> layers;
  std::map<std::string, bool> loaded;
  bool folded = false;        // LayerW::*_wf / *_cs / *_bf are current
  float* stage = nullptr;     // fp32 staging for uploads
  size_t stage_elems = 0;

  // workspace (sized for cfg.max_batch crops)
  void* a_patch = nullptr;
  void* x = nullptr;          // residual stream [B*L, C] of type xdt
  void *xn = nullptr, *qkv = nullptr, *att = nullptr, *hbuf = nullptr;
  float* y = nullptr;
  float* rowstat = nullptr;   // [B*L, 2] LayerNorm (rstd, -mean*rstd) of the residual rows
  float* rowpart = nullptr;   // [B*L, 16, 2] (sum, sum^2) slices handed from GEMM to GEMM
  void* zero_mask = nullptr;  // [B, L-1] 16-bit zeros: the CLS rows of the last block mask nothing
  void* unpad = nullptr;      // dense 16-bit copy of a SMALL padded-layout pass (patch_embed; grown on demand)
  size_t unpad_cap = 0;
  bool stat_fused = false;    // this pass: statistics via rowpart (else the rowstat kernel)
  int nparts = 0;             // valid slices per row in rowpart (1 after embed, width/64 after a GEMM)
  float* e32 = nullptr;       // [head_rows, embed] fp32 head projection
  void* yn = nullptr;         // [head_rows, C] 16-bit: ln_post output (head input)
  int head_rows = 0;          // rows the head buffers (y, yn, e32) hold: the most sequences one pass encodes

  // resample scratch (grown on demand)
  ResampleJob* rs_jobs = nullptr;
  int32_t* rs_coef = nullptr;
  int32_t* rs_bounds = nullptr;
  uint8_t* rs_temp = nullptr;
  size_t rs_jobs_cap = 0, rs_coef_cap = 0, rs_bounds_cap = 0, rs_temp_cap = 0;
  // pinned staging ring for the job descriptors: the upload needs no host-side wait for the stream
  static constexpr int kJobRing = 32;  // (a 6-level blocks flush makes 13 uploads: no slot is reused within a call)
  void* rs_stage[kJobRing] = {};
  size_t rs_stage_cap[kJobRing] = {};
  hipEvent_t rs_stage_done[kJobRing] = {};
  int rs_stage_next = 0;
  // oake_blocks_batch: crop descriptors and the pyramid levels >= 1 of a flush of images
  CropJob* crop_jobs = nullptr;
  uint8_t* pyr = nullptr;
  size_t crop_jobs_cap = 0, pyr_cap = 0;

  // JPEG decode scratch (grown on demand): pinned host coefficients, device coefficients + planes
  int16_t* jp_host = nullptr;
  int16_t* jp_coefs = nullptr;
  uint8_t* jp_planes = nullptr;
  size_t jp_host_cap = 0, jp_coefs_cap = 0, jp_planes_cap = 0;
  hipEvent_t jp_copied = nullptr;  // the last upload out of jp_host has completed

  // profiler (prof_stride > 1: only every prof_stride-th launch is stamped — a stamped launch ends with the
  // runtime's completion signal and cache write-back, which the NEXT kernel pays for; sampled sparsely, a
  // stamped kernel runs behind un-instrumented predecessors, as in the throughput measurement)
  bool prof = false;
  int prof_stride = 1;
  int64_t prof_seq = 0;
  std::vector<ProfSlot> slots;
  std::vector<PendingEvt> pending;
  std::vector<hipEvent_t> evt_pool;
};

namespace {

#define HIP_TRY(h, expr)                                                                      \
  do {                                                                                        \
    hipError_t _e = (expr);                                                                   \
    if (_e != hipSuccess) {                                                                   \
      (h)->err = std::string(#expr) + ": " + hipGetErrorString(_e);                           \
      return OAKE_ERR_HIP;                                                                    \
    }                                                                                         \
  } while (0)

size_t e16() { return 2; }

int fail(oake_handle* h, int code, const std::string& msg) {
  h->err = msg;
  return code;
}

int slot_of(oake_handle* h, const char* name) {
  for (size_t i = 0; i < h->slots.size(); ++i)
    if (h->slots[i].name == name) return (int)i;
  ProfSlot s;
  s.name = name;
  h->slots.push_back(s);
  return (int)h->slots.size() - 1;
}

hipEvent_t get_evt(oake_handle* h) {
  if (!h->evt_pool.empty()) {
    hipEvent_t e = h->evt_pool.back();
    h->evt_pool.pop_back();
    return e;
  }
  hipEvent_t e;
  (void)hipEventCreate(&e);
  return e;
}

// RAII-less bracket: begin returns the index into pending (or -1 when profiling is off)
bool prof_take(oake_handle* h, int sl) {
  h->slots[sl].seen += 1;
  return h->prof_seq++ % h->prof_stride == 0;
}

int prof_begin(oake_handle* h, const char* name, double flops, double bytes, hipStream_t s) {
  if (!h->prof) return -1;
  const int sl = slot_of(h, name);
  if (!prof_take(h, sl)) return -1;
  h->slots[sl].flops += flops;
  h->slots[sl].bytes += bytes;
  h->slots[sl].launches += 1;
  PendingEvt p{sl, get_evt(h), get_evt(h)};
  (void)hipEventRecord(p.a, s);
  h->pending.push_back(p);
  return (int)h->pending.size() - 1;
}
void prof_end(oake_handle* h, int idx, hipStream_t s) {
  if (idx >= 0) (void)hipEventRecord(h->pending[idx].b, s);
}
// Single-kernel launches (GEMMs, attention): the kernel's own begin / end stamps, see common.h
int prof_begin_kernel(oake_handle* h, const char* name, double flops, double bytes) {
  if (!h->prof) return -1;
  const int sl = slot_of(h, name);
  if (!prof_take(h, sl)) return -1;
  h->slots[sl].flops += flops;
  h->slots[sl].bytes += bytes;
  h->slots[sl].launches += 1;
  PendingEvt p{sl, get_evt(h), get_evt(h)};
  h->pending.push_back(p);
  oake::g_launch_start = p.a;
  oake::g_launch_stop = p.b;
  return (int)h->pending.size() - 1;
}
void prof_end_kernel() {
  oake::g_launch_start = nullptr;
  oake::g_launch_stop = nullptr;
}

void prof_collect(oake_handle* h) {
  for (auto& p : h->pending) {
    (void)hipEventSynchronize(p.b);
    float ms = 0.f;
    if (hipEventElapsedTime(&ms, p.a, p.b) == hipSuccess) h->slots[p.slot].ms += ms;
    h->evt_pool.push_back(p.a);
    h->evt_pool.push_back(p.b);
  }
  h->pending.clear();
}

#define RUNK(h, s, name, flops, bytes, call)                \
  do {                                                      \
    (void)prof_begin_kernel(h, name, flops, bytes);         \
    hipError_t _e = (call);                                 \
    prof_end_kernel();                                      \
    if (_e != hipSuccess) {                                 \
      (h)->err = std::string(name) + ": " + hipGetErrorString(_e); \
      return OAKE_ERR_HIP;                                  \
    }                                                       \
  } while (0)

#define RUN(h, s, name, flops, bytes, call)                 \
  do {                                                      \
    const int _pi = prof_begin(h, name, flops, bytes, s);   \
    hipError_t _e = (call);                                 \
    prof_end(h, _pi, s);                                    \
    if (_e != hipSuccess) {                                 \
      (h)->err = std::string(name) + ": " + hipGetErrorString(_e); \
      return OAKE_ERR_HIP;                                  \
    }                                                       \
  } while (0)

int alloc(oake_handle* h, void** p, size_t bytes) {
  HIP_TRY(h, hipMalloc(p, bytes ? bytes : 16));
  return OAKE_OK;
}

const char* kGlobalNames[] = {"visual.conv1.weight",   "visual.class_embedding",
                              "visual.positional_embedding", "visual.ln_pre.weight",
                              "visual.ln_pre.bias",    "visual.ln_post.weight",
                              "visual.ln_post.bias",   "visual.proj"};
const char* kLayerNames[] = {"ln_1.weight",          "ln_1.bias",         "ln_2.weight",
                             "ln_2.bias",            "attn.in_proj_weight", "attn.in_proj_bias",
                             "attn.out_proj.weight", "attn.out_proj.bias", "mlp.c_fc.weight",
                             "mlp.c_fc.bias",        "mlp.c_proj.weight", "mlp.c_proj.bias"};

const char* const kTextGlobalNames[] = {"token_embedding.weight", "positional_embedding", "ln_final.weight",
                                        "ln_final.bias", "text_projection"};

std::string layer_key(int l, const char* leaf, bool text = false) {
  return std::string(text ? "" : "visual.") + "transformer.resblocks." + std::to_string(l) + "." + leaf;
}

int upload_f32(oake_handle* h, float* dst, const float* src, size_t numel) {
  HIP_TRY(h, hipMemcpy(dst, src, numel * sizeof(float), hipMemcpyHostToDevice));
  return OAKE_OK;
}

int upload_16(oake_handle* h, void* dst, const float* src, size_t numel) {
  if (numel > h->stage_elems) return fail(h, OAKE_ERR_INVALID, "staging buffer too small");
  HIP_TRY(h, hipMemcpy(h->stage, src, numel * sizeof(float), hipMemcpyHostToDevice));
  HIP_TRY(h, launch_cast_f32_to_16(h->dt16, h->stage, dst, numel, 1.0f, 0));
  HIP_TRY(h, hipStreamSynchronize(0));
  return OAKE_OK;
}

}  // namespace

int oake::fail_without_handle(int code, const char* text) noexcept {
  try {
    g_create_error = text;
  } catch (...) {  // (out of memory: the status says enough)
  }
  return code;
}

extern "C" {

uint32_t oake_abi_version(void) { return OAKE_ABI_VERSION; }

void oake_default_config(oake_config* c) {
  if (!c) return;
  std::memset(c, 0, sizeof(*c));
  c->image_size = 224;
  c->patch_size = 32;
  c->stride = 32;
  c->padding = 0;
  c->width = 768;
  c->layers = 12;
  c->heads = 12;
  c->mlp_dim = 3072;
  c->embed_dim = 512;
  c->compute_dtype = OAKE_F16;
  c->max_batch = 256;
  c->residual_dtype = OAKE_F16;
}

const char* oake_last_error(const oake_handle* h) {
  return h ? h->err.c_str() : g_create_error.c_str();
}

int oake_grid(const oake_handle* h) { return h ? h->grid : 0; }
int oake_tokens(const oake_handle* h) { return h ? h->tokens : 0; }

void oake_destroy(oake_handle* h) {
  if (!h) return;
  (void)hipSetDevice(h->device);
  (void)hipDeviceSynchronize();
  void* ptrs[] = {h->conv_w, h->cls, h->pos, h->lnpre_g, h->lnpre_b, h->lnpost_g, h->lnpost_b,
                  h->proj, h->stage, h->a_patch, h->x, h->xn, h->qkv, h->att, h->hbuf, h->y, h->e32,
                  h->yn, h->rs_jobs, h->rs_coef, h->rs_bounds, h->rs_temp, h->crop_jobs, h->pyr,
                  h->rowstat, h->rowpart, h->zero_mask, h->unpad, h->jp_coefs, h->jp_planes, h->tok_emb};
  for (void* p : ptrs)
    if (p) (void)hipFree(p);
  for (auto& l : h->layers) {
    void* lp[] = {l.ln1_g, l.ln1_b, l.ln2_g, l.ln2_b, l.in_w, l.out_w, l.fc_w, l.proj_w,
                  l.in_b, l.out_b, l.fc_b, l.proj_b, l.in_w32, l.fc_w32, l.in_wf, l.fc_wf,
                  l.in_cs, l.fc_cs, l.in_bf, l.fc_bf, l.out_wp, l.in_wfp, l.in_csp, l.in_bfp};
    for (void* p : lp)
      if (p) (void)hipFree(p);
  }
  for (int i = 0; i < oake_handle::kJobRing; ++i) {
    if (h->rs_stage[i]) (void)hipHostFree(h->rs_stage[i]);
    if (h->rs_stage_done[i]) (void)hipEventDestroy(h->rs_stage_done[i]);
  }
  if (h->jp_host) (void)hipHostFree(h->jp_host);
  if (h->jp_copied) (void)hipEventDestroy(h->jp_copied);
  prof_collect(h);
  for (auto e : h->evt_pool) (void)hipEventDestroy(e);
  delete h;
}

}  // extern "C"

namespace {

// text != 0: cfg.image_size carries the context length, vocab the vocabulary size; no patch embedding
int create_impl(const oake_config* cfg, int device, oake_handle** out, bool text, int vocab) {
  if (!cfg || !out) {
    g_create_error = "null argument";
    return OAKE_ERR_INVALID;
  }
  *out = nullptr;
  oake_config c = *cfg;
  auto bad = [&](const char* m) {
    g_create_error = m;
    return OAKE_ERR_INVALID;
  };
  if (text) {
    if (c.image_size <= 0 || vocab <= 0) return bad("context and vocab must be positive");
    c.patch_size = 8;  // unused; keeps the geometry checks below meaningful for the vision tower only
    c.stride = 8;
    c.padding = 0;
  }
  if (c.width <= 0 || c.heads <= 0 || c.width != c.heads * 64)
    return bad("width must equal heads * 64 (head_dim 64)");
  if (c.width % 64 != 0 || c.mlp_dim % 64 != 0 || c.width > 1024)
    return bad("width/mlp_dim must be multiples of 64 and width <= 1024");
  if (!text && (c.patch_size % 8 != 0 || (3 * c.patch_size * c.patch_size) % 64 != 0))
    return bad("patch_size must be a multiple of 8");
  if (!text && (c.stride <= 0 || c.padding < 0 || c.image_size + 2 * c.padding < c.patch_size))
    return bad("bad conv1 geometry");
  if (c.embed_dim % 4 != 0 || c.embed_dim > 1024 || c.embed_dim <= 0)
    return bad("embed_dim must be a multiple of 4 and <= 1024");
  if (c.compute_dtype != OAKE_F16 && c.compute_dtype != OAKE_BF16)
    return bad("compute_dtype must be OAKE_F16 or OAKE_BF16");
  if (c.layers <= 0 || c.max_batch <= 0) return bad("layers and max_batch must be positive");
  if (c.residual_dtype != OAKE_F32 && c.residual_dtype != c.compute_dtype)
    return bad("residual_dtype must be OAKE_F32 or equal to compute_dtype");

  hipError_t e = hipSetDevice(device);
  if (e != hipSuccess) {
    g_create_error = std::string("hipSetDevice: ") + hipGetErrorString(e);
    return OAKE_ERR_HIP;
  }
  oake_handle* h = new oake_handle();
  h->cfg = c;
  h->device = device;
  h->dt16 = c.compute_dtype;
  h->xdt = c.residual_dtype == OAKE_F32 ? DT_F32 : c.compute_dtype;
  h->text = text;
  h->vocab = vocab;
  if (text) {
    h->tokens = c.image_size;  // context length
  } else {
    h->grid = (c.image_size + 2 * c.padding - c.patch_size) / c.stride + 1;
    h->p2 = h->grid * h->grid;
    h->tokens = h->p2 + 1;
    h->kpatch = 3 * c.patch_size * c.patch_size;
  }
  h->layers.resize(c.layers);
  if (!text) {
    // Crops per internal pass: at most cfg.max_batch, and at most what keeps a pass at ~25 600 token rows — the size
    // at which a pass's activations (x, qkv, att, hbuf: 12 KB per row) still turn over inside the 256-MB Infinity
    // Cache between the kernel that writes them and the one that reads them.  Measured in one session
    // (tools/mb_sweep.sh, profiles/r04/pass_rows_sweep.log): objects mode (L = 197) 25.4 / 26.0 / 26.2 k crops/s at
    // 512 / 256 / 128 crops per pass, blocks mode (L = 50) 111.0 / 108.3 / 98.4 k at 512 / 256 / 128 and 108.5 /
    // 105.9 at 1024 / 1728 (round 3) — both best at ~25 k rows.
    // cfg.pass_rows names the target (0: this default; < 0: no row cap).  No environment variable is read here: the
    // pass size decides output rounding, and an ABI library takes such things through its arguments (the Python host
    // maps OAKE_PASS_ROWS / OAKE_PASS_CROPS onto the config, oadp_amd/clip/model.py).
    const long rows = c.pass_rows == 0 ? 25600 : c.pass_rows;
    if (rows > 0) {
      const long per = std::max<long>(32, rows / h->tokens / 32 * 32);
      if (per < c.max_batch) h->cfg.max_batch = c.max_batch = (int)per;
    }
  }

  h->pass_cap = c.max_batch;
  const size_t C = c.width, F = c.mlp_dim, E = c.embed_dim, L = h->tokens, B = c.max_batch;
  int rc = OAKE_OK;
  auto A = [&](void** p, size_t bytes) {
    if (rc == OAKE_OK) rc = alloc(h, p, bytes);
  };
  if (text) {
    A((void**)&h->tok_emb, (size_t)vocab * C * 4);
  } else {
    A(&h->conv_w, C * h->kpatch * e16());
    A((void**)&h->cls, C * 4);
    A((void**)&h->lnpre_g, C * 4);
    A((void**)&h->lnpre_b, C * 4);
  }
  A((void**)&h->pos, L * C * 4);
  A((void**)&h->lnpost_g, C * 4);
  A((void**)&h->lnpost_b, C * 4);
  A(&h->proj, C * E * e16());
  for (auto& l : h->layers) {
    A((void**)&l.ln1_g, C * 4);
    A((void**)&l.ln1_b, C * 4);
    A((void**)&l.ln2_g, C * 4);
    A((void**)&l.ln2_b, C * 4);
    A(&l.in_w, 3 * C * C * e16());
    A(&l.out_w, C * C * e16());
    A(&l.fc_w, F * C * e16());
    A(&l.proj_w, C * F * e16());
    A((void**)&l.in_b, 3 * C * 4);
    A((void**)&l.out_b, C * 4);
    A((void**)&l.fc_b, F * 4);
    A((void**)&l.proj_b, C * 4);
    if (h->xdt != DT_F32) {
      A((void**)&l.in_w32, 3 * C * C * 4);
      A((void**)&l.fc_w32, F * C * 4);
      A(&l.in_wf, 3 * C * C * e16());
      A(&l.fc_wf, F * C * e16());
      A((void**)&l.in_cs, 3 * C * 4);
      A((void**)&l.fc_cs, F * 4);
      A((void**)&l.in_bf, 3 * C * 4);
      A((void**)&l.fc_bf, F * 4);
    }
  }
  // (every tensor that goes through the fp32 staging buffer: conv1, c_fc / c_proj, in_proj, the positional
  // embedding and the output projection — C x E exceeds the others on a narrow tower with a wide embedding)
  h->stage_elems = std::max<size_t>(std::max<size_t>(C * h->kpatch, F * C),
                                    std::max<size_t>(std::max<size_t>(3 * C * C, L * C), C * E));
  A((void**)&h->stage, h->stage_elems * 4);
  // workspace
  if (!text) A(&h->a_patch, B * h->p2 * h->kpatch * e16());
  // (+ B rows: in objects mode the object-token stream rides as rows B*L .. B*L+B of the same matrices)
  const size_t R = B * L + B;
  A(&h->x, R * C * (h->xdt == DT_F32 ? 4 : 2));
  A(&h->xn, R * C * e16());
  A(&h->qkv, R * 3 * C * e16());
  A(&h->att, R * C * e16());
  A(&h->hbuf, R * F * e16());
  // vision: one row per crop.  text: sequences shorter than the context pack more than max_batch per
  // pass (oake_encode_text), up to this many — the head buffers must hold them all
  h->head_rows = (int)(text ? B * 4 : B);
  const size_t HR = (size_t)h->head_rows;
  A((void**)&h->y, HR * C * 4);
  A((void**)&h->rowstat, (R + 2) * 2 * 4);
  A((void**)&h->rowpart, R * 32 * 4);
  A(&h->zero_mask, B * (L > 1 ? L - 1 : 1) * 2);  // "nothing masked" for the CLS rows of the last block
  if (rc == OAKE_OK && hipMemset(h->zero_mask, 0, B * (L > 1 ? L - 1 : 1) * 2) != hipSuccess) rc = OAKE_ERR_HIP;
  A((void**)&h->e32, HR * E * 4);
  A(&h->yn, HR * C * e16());
  if (rc != OAKE_OK) {
    g_create_error = h->err;
    oake_destroy(h);
    return rc;
  }
  if (text)
    for (const char* n : kTextGlobalNames) h->loaded[n] = false;
  else
    for (const char* n : kGlobalNames) h->loaded[n] = false;
  for (int l = 0; l < c.layers; ++l)
    for (const char* n : kLayerNames) h->loaded[layer_key(l, n, text)] = false;
  *out = h;
  return OAKE_OK;
}

}  // namespace

extern "C" {

int oake_create(const oake_config* cfg, int device, oake_handle** out) {
  return create_impl(cfg, device, out, false, 0);
}

void oake_text_default_config(oake_text_config* c) {
  if (!c) return;
  std::memset(c, 0, sizeof(*c));
  c->context = 77;
  c->vocab = 49408;
  c->width = 512;
  c->layers = 12;
  c->heads = 8;
  c->mlp_dim = 2048;
  c->embed_dim = 512;
  c->compute_dtype = OAKE_F16;
  c->max_batch = 1024;
}

int oake_text_create(const oake_text_config* tc, int device, oake_handle** out) {
  if (!tc || !out) {
    g_create_error = "null argument";
    return OAKE_ERR_INVALID;
  }
  oake_config c;
  std::memset(&c, 0, sizeof(c));
  c.image_size = tc->context;
  c.width = tc->width;
  c.layers = tc->layers;
  c.heads = tc->heads;
  c.mlp_dim = tc->mlp_dim;
  c.embed_dim = tc->embed_dim;
  c.compute_dtype = tc->compute_dtype;
  c.max_batch = tc->max_batch;
  c.residual_dtype = tc->compute_dtype;
  return create_impl(&c, device, out, true, tc->vocab);
}

int oake_missing_tensors(const oake_handle* h) {
  if (!h) return -1;
  int m = 0;
  for (auto& kv : h->loaded) m += kv.second ? 0 : 1;
  return m;
}

int oake_load_tensor(oake_handle* h, const char* name, const float* data, size_t numel) {
  if (!h || !name || !data) return OAKE_ERR_INVALID;
  HIP_TRY(h, hipSetDevice(h->device));
  const std::string key(name);
  auto it = h->loaded.find(key);
  if (it == h->loaded.end()) return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "unknown tensor: " + key);
  const size_t C = h->cfg.width, F = h->cfg.mlp_dim, E = h->cfg.embed_dim, L = h->tokens;
  auto expect = [&](size_t n) -> int {
    if (numel != n)
      return fail(h, OAKE_ERR_INVALID,
                  key + ": expected " + std::to_string(n) + " elements, got " + std::to_string(numel));
    return OAKE_OK;
  };
  int rc = OAKE_OK;
#define F32(dst, n)                                   \
  do {                                                \
    if ((rc = expect(n)) != OAKE_OK) return rc;       \
    if ((rc = upload_f32(h, dst, data, n)) != OAKE_OK) return rc; \
  } while (0)
#define W16(dst, n)                                   \
  do {                                                \
    if ((rc = expect(n)) != OAKE_OK) return rc;       \
    if ((rc = upload_16(h, dst, data, n)) != OAKE_OK) return rc;  \
  } while (0)

  auto load_proj = [&]() -> int {
    // state_dict layout is [width, embed] (x @ proj); the GEMM wants W[N = embed][K = width]
    if ((rc = expect(C * E)) != OAKE_OK) return rc;
    std::vector<float> t(C * E);
    for (size_t cc = 0; cc < C; ++cc)
      for (size_t ee = 0; ee < E; ++ee) t[ee * C + cc] = data[cc * E + ee];
    return upload_16(h, h->proj, t.data(), C * E);
  };
  if (h->text && key == "token_embedding.weight") F32(h->tok_emb, (size_t)h->vocab * C);
  else if (h->text && key == "positional_embedding") F32(h->pos, L * C);
  else if (h->text && key == "ln_final.weight") F32(h->lnpost_g, C);
  else if (h->text && key == "ln_final.bias") F32(h->lnpost_b, C);
  else if (h->text && key == "text_projection") {
    if ((rc = load_proj()) != OAKE_OK) return rc;
  }
  else if (key == "visual.conv1.weight") W16(h->conv_w, C * h->kpatch);
  else if (key == "visual.class_embedding") F32(h->cls, C);
  else if (key == "visual.positional_embedding") F32(h->pos, L * C);
  else if (key == "visual.ln_pre.weight") F32(h->lnpre_g, C);
  else if (key == "visual.ln_pre.bias") F32(h->lnpre_b, C);
  else if (key == "visual.ln_post.weight") F32(h->lnpost_g, C);
  else if (key == "visual.ln_post.bias") F32(h->lnpost_b, C);
  else if (key == "visual.proj") {
    // state_dict layout is [width, embed] (x @ proj); the GEMM wants W[N = embed][K = width]
    if ((rc = expect(C * E)) != OAKE_OK) return rc;
    std::vector<float> t(C * E);
    for (size_t cc = 0; cc < C; ++cc)
      for (size_t ee = 0; ee < E; ++ee) t[ee * C + cc] = data[cc * E + ee];
    if ((rc = upload_16(h, h->proj, t.data(), C * E)) != OAKE_OK) return rc;
  }
  else {
    // visual.transformer.resblocks.<l>.<leaf>
    const std::string prefix = h->text ? "transformer.resblocks." : "visual.transformer.resblocks.";
    const size_t dot = key.find('.', prefix.size());
    const int l = std::stoi(key.substr(prefix.size(), dot - prefix.size()));
    const std::string leaf = key.substr(dot + 1);
    LayerW& w = h->layers[l];
    if (leaf == "ln_1.weight") F32(w.ln1_g, C);
    else if (leaf == "ln_1.bias") F32(w.ln1_b, C);
    else if (leaf == "ln_2.weight") F32(w.ln2_g, C);
    else if (leaf == "ln_2.bias") F32(w.ln2_b, C);
    else if (leaf == "attn.in_proj_weight") {
      // fold the attention scale head_dim^-0.5 = 1/8 (exact in binary) into the q rows
      if ((rc = expect(3 * C * C)) != OAKE_OK) return rc;
      HIP_TRY(h, hipMemcpy(h->stage, data, numel * 4, hipMemcpyHostToDevice));
      HIP_TRY(h, launch_scale_f32(h->stage, C * C, 0.125f, 0));
      HIP_TRY(h, launch_cast_f32_to_16(h->dt16, h->stage, w.in_w, numel, 1.0f, 0));
      if (w.in_w32) HIP_TRY(h, hipMemcpyAsync(w.in_w32, h->stage, numel * 4, hipMemcpyDeviceToDevice, 0));
      HIP_TRY(h, hipStreamSynchronize(0));
    } else if (leaf == "attn.in_proj_bias") {
      F32(w.in_b, 3 * C);
      HIP_TRY(h, launch_scale_f32(w.in_b, C, 0.125f, 0));
      HIP_TRY(h, hipStreamSynchronize(0));
    } else if (leaf == "attn.out_proj.weight") {
      W16(w.out_w, C * C);
#if OAKE_LAB
      // (a reload after OAKE_OPT_FUSE_ATTN_OUT was switched on: attn_out_kernel's fragment-order copy follows the weight)
      if (w.out_wp) {
        HIP_TRY(h, launch_permute_out_w(h->dt16, w.out_w, w.out_wp, 0));
        HIP_TRY(h, hipStreamSynchronize(0));
      }
#endif
    }
    else if (leaf == "attn.out_proj.bias") F32(w.out_b, C);
    else if (leaf == "mlp.c_fc.weight") {
      W16(w.fc_w, F * C);
      if (w.fc_w32) HIP_TRY(h, hipMemcpy(w.fc_w32, data, numel * 4, hipMemcpyHostToDevice));
    }
    else if (leaf == "mlp.c_fc.bias") F32(w.fc_b, F);
    else if (leaf == "mlp.c_proj.weight") W16(w.proj_w, C * F);
    else if (leaf == "mlp.c_proj.bias") F32(w.proj_b, C);
    else return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "unknown tensor: " + key);
  }
#undef F32
#undef W16
  it->second = true;
  h->folded = false;
  return OAKE_OK;
}

}  // extern "C"

namespace {

// ---- shared pieces of the two schedules -------------------------------------------------------
// row0: first residual row the call works on (offsets the row-statistics buffers); A / out already
// point at that row.
int gemm(oake_handle* h, hipStream_t s, const char* name, int epi, const void* A, const void* W,
         const float* bias, void* out, int M, int N, int K, int ldo,
         const float* rowstat = nullptr, const float* colsum = nullptr, size_t row0 = 0,
         int nparts_in = 0) {
  GemmArgs a{};
  a.A = A; a.W = W; a.bias = bias; a.out = out; a.M = M; a.N = N; a.K = K; a.ldo = ldo;
  a.rowstat = rowstat ? rowstat + row0 * 2 : nullptr;
  a.colsum = colsum;
  a.opts = &h->opts;
  // Which kernel runs is decided per call, from the shape actually passed (the persistent kernel takes
  // LayerNorm statistics as per-row (sum, sum^2) slices, the small kernels as (rstd, -mean rstd)):
  // ln_stats() prepared whichever this call needs and returned nparts_in.
  const bool persistent = gemm_uses_persistent(M, N, K, &h->opts);
  float* part = h->rowpart + row0 * 32;
  if ((epi == EPI_T16_BIAS_LN || epi == EPI_T16_GELU_LN) && persistent) {
    if (nparts_in < 1) return fail(h, OAKE_ERR_STATE, std::string(name) + ": no row statistics for the persistent kernel");
    a.rowpart_in = part;
    a.nparts = nparts_in;
  }
  // row statistics travel GEMM -> GEMM when the stream's shapes run the persistent kernel
  const char* xb = reinterpret_cast<const char*>(h->x);
  const bool to_resid = out == xb + row0 * (size_t)ldo * (h->xdt == DT_F32 ? 4 : 2);
  if (h->stat_fused && epi == EPI_RESID16 && to_resid) {
    if (!persistent)  // (stat_fused promises the next LN-folded GEMM a hand-over; only the persistent kernel writes one)
      return fail(h, OAKE_ERR_STATE, std::string(name) + ": statistics hand-over needs the persistent kernel");
    a.rowpart_out = part;
  }
  RUNK(h, s, name, 2.0 * M * N * K, 0.0, launch_gemm(h->dt16, epi, a, s));
  if (a.rowpart_out) h->nparts = N / 64;
  return OAKE_OK;
}

// LayerNorm statistics of residual rows [r0, r0 + M) (xr points at row r0) for the LN-folded GEMM
// [M, N, K] that follows.  Returns through *nparts what gemm() needs: > 0 = the persistent kernel reads
// that many (sum, sum^2) slices per row from rowpart — handed over by the kernel that wrote the rows
// (stat_fused) or produced here by one rowsums pass (slot 0); 0 = a small kernel reads (rstd, -mean rstd)
// from rowstat, produced here.
int ln_stats(oake_handle* h, hipStream_t s, const char* xr, size_t r0, int M, int N, int K, int* nparts) {
  if (gemm_uses_persistent(M, N, K, &h->opts)) {
    if (h->stat_fused) {
      *nparts = h->nparts;
      return OAKE_OK;
    }
    RUN(h, s, "rowsums", 0.0, (double)M * K * 2,
        launch_rowsums(xr, h->xdt, K, h->rowpart + r0 * 32, M, K, s));
    *nparts = 1;
    return OAKE_OK;
  }
  if (h->stat_fused)  // (cannot happen with the current kernel selection: stat_fused implies M > 1024)
    return fail(h, OAKE_ERR_STATE, "statistics hand-over into a non-persistent GEMM");
  RUN(h, s, "rowstat", 0.0, (double)M * K * 2, launch_rowstat(xr, h->xdt, K, h->rowstat + r0 * 2, M, K, s));
  *nparts = 0;
  return OAKE_OK;
}

// the zero-padded 16-bit batch conv1 gathers its patches from when the convolution pads or its stride cuts patches
// (objects mode): hp rows of ws pixels per colour plane, the image at (padding, padding)
bool padded_geometry(const oake_handle* h, int* pad, int* hp, int* ws) {
  const oake_config& c = h->cfg;
  if (h->text || (c.stride == c.patch_size && c.padding == 0)) return false;
  *pad = c.padding;
  *hp = c.image_size + 2 * c.padding;
  *ws = (c.image_size + 2 * c.padding + 7) & ~7;
  return h->patch_direct && h->xdt != DT_F32 && (h->grid - 1) * c.stride + c.patch_size <= *hp &&
         (size_t)3 * *hp * *ws <= (size_t)h->p2 * h->kpatch && c.image_size % 4 == 0;
}

// in_padded: `imgs` IS that padded batch already (OAKE_LAYOUT_PADDED: the crops were written into it by
// oake_crop_resize_normalize_batch) — no pad pass
int patch_embed(oake_handle* h, hipStream_t s, const void* imgs, int in_dtype, int nb, bool in_padded = false) {
  const oake_config& c = h->cfg;
  const int C = c.width, L = h->tokens;
  const size_t in_es = in_dtype == DT_F32 ? 4 : 2;
  GemmArgs a{};
  a.W = h->conv_w; a.bias = nullptr; a.out = h->x;
  a.M = nb * h->p2; a.N = C; a.K = h->kpatch; a.ldo = C; a.pos = h->pos; a.P2 = h->p2; a.L = L;
  a.opts = &h->opts;
  // Images already in the compute type (the reference casts to model.dtype before conv1; the device
  // preprocessing writes fp16 crops): the conv1 GEMM's DMA waves gather the patch rows straight from the
  // NCHW batch — no im2col pass, no a_patch round trip.  Other inputs (fp32, the other 16-bit type,
  // strides that cut patches: objects mode) go through im2col, which also does the cast.
  const bool direct = !in_padded && h->patch_direct && in_dtype == h->dt16 && h->xdt != DT_F32 &&
                      gemm_patch_direct_ok(c.image_size, c.patch_size, c.stride, c.padding, a.M, a.N, a.K, &h->opts) &&
                      reinterpret_cast<uintptr_t>(imgs) % 16 == 0;
  // ... and where the convolution pads or its stride cuts patches (objects mode: stride 16, padding 15), from a
  // zero-padded 16-bit copy of the batch in the a_patch buffer: a third of the im2col matrix's bytes, written
  // once, the overlapping patches re-read from the L2
  const int hp = c.image_size + 2 * c.padding;             // rows per padded plane
  const int ws = (c.image_size + 2 * c.padding + 7) & ~7;  // padded row stride (pixels)
  const bool padded = !direct && h->patch_direct && h->xdt != DT_F32 &&
                      (c.stride != c.patch_size || c.padding != 0) &&  // (plain geometry, other input type: im2col is the cheaper cast)
                      gemm_patch_padded_ok(c.patch_size, c.stride, a.M, a.N, a.K, &h->opts) &&
                      (h->grid - 1) * c.stride + c.patch_size <= hp &&
                      (size_t)3 * hp * ws <= (size_t)h->p2 * h->kpatch;  // fits the im2col buffer
  // fp32 images in the plain geometry (what the reference hands over, globals.py:54-57): the same gather, with
  // the cast done by the GEMM's DMA waves on the way into LDS — no im2col pass either.  Opt-in (patch_direct = 2):
  // measured, the register-staged A path makes conv1 97.8 us against 60.5 + 43.2 for GEMM + im2col — +0.3 % on one
  // lane, but -0.6 % with two lanes (the DMA waves' ordinary loads and ds_writes cost the partner lane more than
  // the im2col pass did), profiles/r03/ab_session_e_*.log
  const bool direct32 = !direct && h->patch_direct >= 2 && in_dtype == DT_F32 && h->xdt != DT_F32 &&
                        gemm_patch_f32_ok(c.image_size, c.patch_size, c.stride, c.padding, a.M, a.N, a.K, &h->opts) &&
                        reinterpret_cast<uintptr_t>(imgs) % 16 == 0;
  if (in_padded && !padded) {
    // a pass too small for the persistent GEMM (a handful of crops): back to a dense batch (a scratch of its own: no
    // workspace buffer is large enough in every geometry) and the im2col route
    const size_t need = (size_t)nb * 3 * c.image_size * c.image_size * 2;
    if (need > h->unpad_cap) {
      HIP_TRY(h, hipStreamSynchronize(s));
      if (h->unpad) HIP_TRY(h, hipFree(h->unpad));
      h->unpad = nullptr; h->unpad_cap = 0;
      HIP_TRY(h, hipMalloc(&h->unpad, need));
      h->unpad_cap = need;
    }
    RUN(h, s, "unpad_nchw", 0.0, 2.0 * need,
        launch_unpad_nchw(imgs, h->unpad, nb, c.image_size, c.padding, hp, ws, s));
    return patch_embed(h, s, h->unpad, h->dt16, nb, false);
  }
  if (direct || direct32) {
    a.A = imgs;
    a.patch_S = c.image_size; a.patch_P = c.patch_size; a.patch_G = h->grid;
    a.patch_f32 = direct32 ? 1 : 0;
  } else if (padded && in_padded) {
    a.A = imgs;
    a.patch_S = ws; a.patch_H = hp; a.patch_P = c.patch_size; a.patch_T = c.stride; a.patch_G = h->grid;
  } else if (padded) {
    RUN(h, s, "pad_nchw", 0.0, (double)nb * 3 * hp * ws * 2 + (double)nb * 3 * c.image_size * c.image_size * in_es,
        launch_pad_nchw(h->dt16, imgs, in_dtype, h->a_patch, nb, c.image_size, c.padding, hp, ws, s));
    a.A = h->a_patch;
    a.patch_S = ws; a.patch_H = hp; a.patch_P = c.patch_size; a.patch_T = c.stride; a.patch_G = h->grid;
  } else {
    const double im_bytes = (double)nb * h->p2 * h->kpatch * 2 + (double)nb * 3 * c.image_size * c.image_size * in_es;
    RUN(h, s, "im2col", 0.0, im_bytes,
        launch_im2col(h->dt16, imgs, in_dtype, h->a_patch, nb, c.image_size, c.patch_size, c.stride,
                      c.padding, h->grid, s));
    a.A = h->a_patch;
  }
  RUNK(h, s, "gemm_conv1", 2.0 * a.M * a.N * a.K, 0.0,
      launch_gemm(h->dt16, h->xdt == DT_F32 ? EPI_PATCH : EPI_PATCH16, a, s));
  // 16-bit residual stream + every main-stream GEMM on the persistent kernel: LayerNorm statistics
  // are produced by the kernel that writes x (here: slot 0) and consumed by the next GEMM
  const int T = nb * L;
  h->cur_len = L;
  h->stat_fused = h->xdt != DT_F32 && C % 64 == 0 && C / 64 <= 16 &&
                  gemm_uses_persistent(T, C, C, &h->opts) && gemm_uses_persistent(T, C, c.mlp_dim, &h->opts) &&
                  gemm_uses_persistent(T, 2 * C, C, &h->opts) && gemm_uses_persistent(T, c.mlp_dim, C, &h->opts);
  RUN(h, s, "embed_ln_pre", 0.0, 2.0 * nb * L * C * 4,
      launch_embed_ln_pre(h->x, h->xdt, h->cls, h->pos, h->lnpre_g, h->lnpre_b, nb, L, C,
                          h->stat_fused ? h->rowpart : nullptr, s));
  h->nparts = 1;
  return OAKE_OK;
}

// ln_1 + in-proj of residual rows [r0, r0 + M) -> the same rows of h->qkv ([., 3C]; kv_only:
// columns C.. only)
int in_proj_rows(oake_handle* h, hipStream_t s, const LayerW& w, size_t r0, int M, bool kv_only,
                 const char* name) {
  const int C = h->cfg.width;
  const int n0 = kv_only ? C : 0, N = 3 * C - n0;
  const size_t es = 2, xs = h->xdt == DT_F32 ? 4 : 2;
  char* out = reinterpret_cast<char*>(h->qkv) + (r0 * 3 * C + n0) * es;
  const char* xr = reinterpret_cast<const char*>(h->x) + r0 * C * xs;
  if (h->xdt == DT_F32) {
    char* xn = reinterpret_cast<char*>(h->xn) + r0 * C * es;
    RUN(h, s, "layernorm", 0.0, (double)M * C * 6,
        launch_layernorm(h->dt16, xr, h->xdt, C, w.ln1_g, w.ln1_b, xn, M, C, s));
    const char* wp = reinterpret_cast<const char*>(w.in_w) + (size_t)n0 * C * es;
    return gemm(h, s, name, EPI_T16_BIAS, xn, wp, w.in_b + n0, out, M, N, C, 3 * C);
  }
  // 16-bit residual stream: ln_1 folded into the GEMM, which reads the raw residual rows
  int np = 0, rc;
  if ((rc = ln_stats(h, s, xr, r0, M, N, C, &np))) return rc;
  const char* wp = reinterpret_cast<const char*>(w.in_wf) + (size_t)n0 * C * es;
  return gemm(h, s, name, EPI_T16_BIAS_LN, xr, wp, w.in_bf + n0, out, M, N, C, 3 * C, h->rowstat,
              w.in_cs + n0, r0, np);
}

// attention out-proj (+residual) -> ln_2 + c_fc (+QuickGELU) -> c_proj (+residual) of rows [r0, r0 + M)
int mlp_rows(oake_handle* h, hipStream_t s, const LayerW& w, size_t r0, int M, const char* sfx,
             bool out_proj_done = false) {
  const int C = h->cfg.width, F = h->cfg.mlp_dim;
  const size_t es = 2, xs = h->xdt == DT_F32 ? 4 : 2;
  char* xr = reinterpret_cast<char*>(h->x) + r0 * C * xs;
  const char* att = reinterpret_cast<const char*>(h->att) + r0 * C * es;
  char* hb = reinterpret_cast<char*>(h->hbuf) + r0 * F * es;
  const std::string n_out = std::string("gemm_out_proj") + sfx, n_fc = std::string("gemm_c_fc") + sfx,
                    n_pr = std::string("gemm_c_proj") + sfx;
  const int resid = h->xdt == DT_F32 ? EPI_RESID : EPI_RESID16;
  int rc;
  if (!out_proj_done &&
      (rc = gemm(h, s, n_out.c_str(), resid, att, w.out_w, w.out_b, xr, M, C, C, C, nullptr, nullptr, r0)))
    return rc;
  if (h->xdt == DT_F32) {
    char* xn = reinterpret_cast<char*>(h->xn) + r0 * C * es;
    RUN(h, s, "layernorm", 0.0, (double)M * C * 6,
        launch_layernorm(h->dt16, xr, h->xdt, C, w.ln2_g, w.ln2_b, xn, M, C, s));
    if ((rc = gemm(h, s, n_fc.c_str(), EPI_T16_GELU, xn, w.fc_w, w.fc_b, hb, M, F, C, F))) return rc;
  } else {
    // ln_2 folded into c_fc: the GEMM reads the raw residual rows
    int np = 0;
    if ((rc = ln_stats(h, s, xr, r0, M, F, C, &np))) return rc;
    if ((rc = gemm(h, s, n_fc.c_str(), EPI_T16_GELU_LN, xr, w.fc_wf, w.fc_bf, hb, M, F, C, F, h->rowstat,
                   w.fc_cs, r0, np)))
      return rc;
  }
  return gemm(h, s, n_pr.c_str(), resid, hb, w.proj_w, w.proj_b, xr, M, C, F, C, nullptr, nullptr, r0);
}

// The three-images-per-160-row-tile form (csrc/qkv_attn.hip) lost its A/B to the four-image form in round 5 and no shipped
// configuration reaches it (51 <= L <= 53 only): it is in liboake_hip_lab.so alone; the product runs such sequence lengths
// through the two launches (LN-folded qkv GEMM + attention kernel).
#if OAKE_LAB
inline bool tri_supported(int L, int heads, int width, int n) { return qkv_attn_supported(L, heads, width, n); }
#else
inline bool tri_supported(int, int, int, int) { return false; }
#endif

// which fused form a handle's geometry takes: the 208-row tile kernel (csrc/qkv_attn_obj.hip: objects mode, or four images
// of <= 50 tokens per tile) or the 160-row one (csrc/qkv_attn.hip: three images of <= 53 tokens; fuse_qkv_attn == 2 asks
// for it where both apply) — they read the folded in-projection in different column orders
bool uses_qkv_attn_quad(const oake_handle* h) {
  return h->fuse_qkv_attn == 1 && qkv_attn_quad_supported(h->tokens, h->cfg.heads, h->cfg.width, 1);
}
bool qkv_perm_is_obj(const oake_handle* h) {
  return qkv_attn_obj_supported(h->tokens, h->cfg.heads, h->cfg.width, 1) || uses_qkv_attn_quad(h);
}

// the head-major copies of the folded in-projection (qkv_attn.hip): made on the first pass that takes the fused path
int ensure_qkv_perm(oake_handle* h) {
  if (h->qkv_perm) return OAKE_OK;
  // (reached from check_ready with the fold already done — the option toggled after the first encode — on whatever device
  // the calling thread last used: the allocations and the permute launches below belong on the handle's)
  HIP_TRY(h, hipSetDevice(h->device));
  const size_t C = h->cfg.width;
  for (auto& w : h->layers) {
    if (!w.in_wfp) HIP_TRY(h, hipMalloc(&w.in_wfp, 3 * C * C * 2));
    if (!w.in_csp) HIP_TRY(h, hipMalloc((void**)&w.in_csp, 3 * C * 4));
    if (!w.in_bfp) HIP_TRY(h, hipMalloc((void**)&w.in_bfp, 3 * C * 4));
    if (qkv_perm_is_obj(h)) {  // (a handle has ONE geometry)
      HIP_TRY(h, launch_permute_qkv_obj(w.in_wf, w.in_bf, w.in_cs, w.in_wfp, w.in_bfp, w.in_csp, (int)C, 0));
    } else {
#if OAKE_LAB
      HIP_TRY(h, launch_permute_qkv(h->dt16, w.in_wf, w.in_bf, w.in_cs, w.in_wfp, w.in_bfp, w.in_csp, (int)C, 0));
#else
      return fail(h, OAKE_ERR_STATE, "qkv_attn: the three-image form is in the lab build only");
#endif
    }
  }
  HIP_TRY(h, hipStreamSynchronize(0));
  h->qkv_perm = true;
  return OAKE_OK;
}

// true when the main token stream of this pass takes ln_1 + in_proj + attention as ONE kernel (qkv_attn.hip)
bool fuses_qkv_attn(const oake_handle* h, int nb) {
  if (!(h->fuse_qkv_attn && h->stat_fused && !h->text && h->xdt != DT_F32)) return false;
  if (uses_qkv_attn_quad(h)) return qkv_attn_quad_supported(h->cur_len, h->cfg.heads, h->cfg.width, nb);
  return !qkv_perm_is_obj(h) && tri_supported(h->cur_len, h->cfg.heads, h->cfg.width, nb);
}

int main_in_proj(oake_handle* h, hipStream_t s, const LayerW& w, int T, bool kv_only) {
  return in_proj_rows(h, s, w, 0, T, kv_only, kv_only ? "gemm_kv" : "gemm_qkv");
}

int main_block_tail(oake_handle* h, hipStream_t s, const LayerW& w, int nb) {
  // attention + out_proj + MLP of the main token stream (qkv already computed)
  const int C = h->cfg.width, L = h->cur_len, T = nb * L;
  const int Lp = L;  // (the profile quotes ALGORITHMIC attention FLOPs, 4 L^2 d per head: padded key / query tiles are not work)
  // L <= 64 on the 16-bit residual stream (encode_image, blocks mode): attention + out_proj + residual + the row
  // statistics of the next LayerNorm in one kernel, one workgroup per image; `att` is never written (attn_out.hip)
#if OAKE_LAB
  if (h->fuse_attn_out && h->stat_fused && !h->text && w.out_wp && attn_out_supported(L, h->cfg.heads, C)) {
    RUNK(h, s, "attn_out", 4.0 * nb * h->cfg.heads * (double)Lp * Lp * 64 + 2.0 * T * C * C, (double)T * 5 * C * 2,
         launch_attn_out(h->dt16, h->qkv, w.out_wp, w.out_b, h->x, h->rowpart, nb, L, s));
    h->nparts = C / 64;
    return mlp_rows(h, s, w, 0, T, "", true);
  }
#endif
  RUNK(h, s, "attention", 4.0 * nb * h->cfg.heads * (double)Lp * Lp * 64, (double)T * 4 * C * 2,
      launch_attention(h->dt16, h->qkv, h->att, nb, L, h->cfg.heads, h->text ? 1 : 0, s, nullptr, nullptr, 0,
                       nullptr, &h->opts));
  return mlp_rows(h, s, w, 0, T, "");
}

// objects mode: ln_1 + in_proj + attention of both streams (a crop's tokens and its object token) as ONE kernel
bool fuses_qkv_attn_obj(const oake_handle* h, int nb) {
  return h->fuse_qkv_attn && h->stat_fused && !h->text && h->xdt != DT_F32 && h->qkv_perm &&
         qkv_attn_obj_supported(h->cur_len, h->cfg.heads, h->cfg.width, nb);
}

// ln_1 + in_proj + attention of the main token stream as one kernel, then out_proj + MLP
int main_qkv_attn(oake_handle* h, hipStream_t s, const LayerW& w, int nb) {
  const int C = h->cfg.width, L = h->cur_len, T = nb * L;
  int np = 0, rc;
  if ((rc = ln_stats(h, s, reinterpret_cast<const char*>(h->x), 0, T, 3 * C, C, &np))) return rc;
  if (np < 1 || !w.in_wfp) return fail(h, OAKE_ERR_STATE, "qkv_attn: no row statistics / permuted weights");
  if (uses_qkv_attn_quad(h) && qkv_attn_quad_supported(L, h->cfg.heads, C, nb)) {
    RUNK(h, s, "qkv_attn", 2.0 * T * 3 * C * C + 4.0 * nb * h->cfg.heads * (double)L * L * 64, 0.0,
         launch_qkv_attn_quad(h->dt16, h->x, w.in_wfp, w.in_bfp, w.in_csp, h->rowpart, np, h->att, nb, L, h->cfg.heads,
                              &h->opts, s, nullptr));
    return mlp_rows(h, s, w, 0, T, "");
  }
#if OAKE_LAB
  RUNK(h, s, "qkv_attn", 2.0 * T * 3 * C * C + 4.0 * nb * h->cfg.heads * (double)L * L * 64, 0.0,
       launch_qkv_attn(h->dt16, h->x, w.in_wfp, w.in_bfp, w.in_csp, h->rowpart, np, h->att, nb, L, h->cfg.heads,
                       &h->opts, s));
  return mlp_rows(h, s, w, 0, T, "");
#else
  return fail(h, OAKE_ERR_STATE, "qkv_attn: the three-image form is in the lab build only");
#endif
}


// ln_post over `nb` rows (x + i*row_stride) -> @ proj -> optional L2 normalise -> out
int head(oake_handle* h, hipStream_t s, const void* x, int x_dtype, long row_stride, void* outp,
         int out_dtype, int normalize, int nb) {
  const int C = h->cfg.width, E = h->cfg.embed_dim;
  RUN(h, s, "head_ln_post", 0.0, (double)nb * C * 6,
      launch_layernorm(h->dt16, x, x_dtype, row_stride, h->lnpost_g, h->lnpost_b, h->yn, nb, C, s));
  int rc;
  if ((rc = gemm(h, s, "gemm_head_proj", EPI_F32_BIAS, h->yn, h->proj, nullptr, h->e32, nb, E, C, E)))
    return rc;
  RUN(h, s, "head_l2norm", 0.0, (double)nb * E * 6,
      launch_l2norm_rows(h->e32, outp, out_dtype, normalize, nb, E, s));
  return OAKE_OK;
}

int check_ready(oake_handle* h) {
  const int m = oake_missing_tensors(h);
  if (m != 0) return fail(h, OAKE_ERR_STATE, std::to_string(m) + " weight tensors not loaded");
  if (!h->folded && h->xdt != DT_F32) {
    const int C = h->cfg.width, F = h->cfg.mlp_dim;
    HIP_TRY(h, hipSetDevice(h->device));
    for (auto& w : h->layers) {
      HIP_TRY(h, launch_fold_ln(h->dt16, w.in_w32, w.ln1_g, w.ln1_b, w.in_b, w.in_wf, w.in_cs, w.in_bf,
                                3 * C, C, 0));
      HIP_TRY(h, launch_fold_ln(h->dt16, w.fc_w32, w.ln2_g, w.ln2_b, w.fc_b, w.fc_wf, w.fc_cs, w.fc_bf,
                                F, C, 0));
    }
    HIP_TRY(h, hipStreamSynchronize(0));
    h->qkv_perm = false;
  }
  h->folded = true;
  if (h->fuse_qkv_attn && !h->text && h->xdt != DT_F32 && !h->qkv_perm &&
      (tri_supported(h->tokens, h->cfg.heads, h->cfg.width, 1) || qkv_perm_is_obj(h)))
    return ensure_qkv_perm(h);
  return OAKE_OK;
}

size_t dtype_size(int dt) { return dt == DT_F32 ? 4 : (dt == DT_U8 ? 1 : 2); }

}  // namespace

namespace {

template <typename P>
int grow(oake_handle* h, hipStream_t s, P** p, size_t* cap, size_t need_bytes) {
  if (need_bytes <= *cap) return OAKE_OK;
  HIP_TRY(h, hipStreamSynchronize(s));
  if (*p) HIP_TRY(h, hipFree(*p));
  *p = nullptr;
  const size_t bytes = need_bytes + need_bytes / 4 + 4096;
  HIP_TRY(h, hipMalloc(reinterpret_cast<void**>(p), bytes));
  *cap = bytes;
  return OAKE_OK;
}

int ksize_for(int in_size, int out_size) {
  if (in_size == out_size) return 1;
  double filterscale = (double)((float)in_size) / out_size;
  if (filterscale < 1.0) filterscale = 1.0;
  return (int)std::ceil(2.0 * filterscale) * 2 + 1;  // Pillow: (int)ceil(support) * 2 + 1
}

// host descriptors -> a pinned ring slot -> device, asynchronously (a wait only if the slot's previous
// upload, kJobRing calls ago, has not executed yet)
int upload_async(oake_handle* h, hipStream_t s, const void* host, size_t bytes, void* d_dst) {
  const int slot = h->rs_stage_next;
  h->rs_stage_next = (slot + 1) % oake_handle::kJobRing;
  if (!h->rs_stage_done[slot])
    HIP_TRY(h, hipEventCreateWithFlags(&h->rs_stage_done[slot], hipEventDisableTiming));
  else
    HIP_TRY(h, hipEventSynchronize(h->rs_stage_done[slot]));
  if (bytes > h->rs_stage_cap[slot]) {
    if (h->rs_stage[slot]) HIP_TRY(h, hipHostFree(h->rs_stage[slot]));
    h->rs_stage[slot] = nullptr;
    h->rs_stage_cap[slot] = 0;
    HIP_TRY(h, hipHostMalloc(&h->rs_stage[slot], bytes * 2, hipHostMallocDefault));
    h->rs_stage_cap[slot] = bytes * 2;
  }
  std::memcpy(h->rs_stage[slot], host, bytes);
  HIP_TRY(h, hipMemcpyAsync(d_dst, h->rs_stage[slot], bytes, hipMemcpyHostToDevice, s));
  HIP_TRY(h, hipEventRecord(h->rs_stage_done[slot], s));
  return OAKE_OK;
}

// jobs (each naming its source image) -> device, scratch sizing, three launches.  The offsets of `jobs`
// are filled here.  out_dtype DT_U8: every job writes its own image to job.u8_out.
int run_resample(oake_handle* h, hipStream_t s, std::vector<ResampleJob>& jobs, int out_size,
                 const float* mean3, const float* std3, void* d_out, int out_dtype, int out_pad = 0, int out_hp = 0,
                 int out_ws = 0) {
  if (jobs.empty()) return OAKE_OK;
  long coef = 0, bnd = 0, temp = 0;
  int max_out = 1;
  long max_ch_rw = 1, max_chq_rw = 1, max_rh_rw = 1;
  for (auto& j : jobs) {
    if (!j.tr && (long)j.ch > 100L * j.cw && j.rh < j.ch) {  // Pillow resamples these vertically first
      std::swap(j.cw, j.ch); std::swap(j.rw, j.rh); std::swap(j.sx0, j.sy0); std::swap(j.cx, j.cy);
      j.tr = 1;
    }
    j.kh = ksize_for(j.cw, j.rw);
    j.kv = ksize_for(j.ch, j.rh);
    j.coefh_off = coef; coef += (long)j.rw * j.kh;
    j.coefv_off = coef; coef += (long)j.rh * j.kv;
    j.boundh_off = bnd; bnd += 2L * j.rw;
    j.boundv_off = bnd; bnd += 2L * j.rh;
    j.tstride = 12 * ((j.rw + 3) / 4);  // rows of the intermediate image: whole 12-byte quads of pixels
    j.temp_off = temp; temp += ((long)j.ch * j.tstride + 15) & ~15L;
    max_out = std::max(max_out, std::max(j.rw, j.rh));
    max_ch_rw = std::max(max_ch_rw, (long)j.ch * j.rw);
    max_chq_rw = std::max(max_chq_rw, (long)((j.ch + 3) / 4) * ((j.rw + 3) & ~3));  // (resample_h_kernel: four rows per thread, whole quads)
    max_rh_rw = std::max(max_rh_rw, (long)j.rh * j.rw);
  }
  if (max_ch_rw > 0x7fffffffL || max_rh_rw > 0x7fffffffL) return fail(h, OAKE_ERR_INVALID, "crop too large");
  int rc;
  if ((rc = grow(h, s, &h->rs_jobs, &h->rs_jobs_cap, jobs.size() * sizeof(ResampleJob)))) return rc;
  // (+ 16: the horizontal pass reads a column's coefficients in groups of four and may touch up to three entries past the
  // last column's row of the table)
  if ((rc = grow(h, s, &h->rs_coef, &h->rs_coef_cap, (size_t)coef * 4 + 16))) return rc;
  if ((rc = grow(h, s, &h->rs_bounds, &h->rs_bounds_cap, (size_t)bnd * 4))) return rc;
  // (+ 16: resample_v4_kernel's 16-byte loads start at the 4-byte-aligned address below a 12-byte window and may
  // read up to 4 bytes past it — past the last job's temp image when the window is its last 12 bytes)
  if ((rc = grow(h, s, &h->rs_temp, &h->rs_temp_cap, (size_t)temp + 16))) return rc;
  if ((rc = upload_async(h, s, jobs.data(), jobs.size() * sizeof(ResampleJob), h->rs_jobs))) return rc;
  double bytes = (double)temp * 2;
  if (out_dtype == DT_U8)
    for (auto& j : jobs) bytes += (double)j.rh * j.rw * 3;
  else
    bytes += (double)jobs.size() * out_size * out_size * 3 * (out_dtype == DT_F32 ? 4 : 2);
  RUN(h, s, "resample", 0.0, bytes,
      launch_resample(h->rs_jobs, (int)jobs.size(), max_out, max_chq_rw, max_rh_rw, h->rs_coef, h->rs_bounds,
                      h->rs_temp, out_size, mean3, std3, d_out, out_dtype, s, out_pad, out_hp, out_ws));
  return OAKE_OK;
}

// `preprocess(image.crop(box))` geometry of one box: PIL Image.crop (every coordinate through Python
// round(), ties to even; zero fill outside), then Resize(out_size, BICUBIC) + CenterCrop, or a squash.
int fill_crop_job(oake_handle* h, ResampleJob& j, const uint8_t* img, int height, int width, const float* box,
                  int out_size, int squash) {
  j = ResampleJob{};
  j.img = img; j.height = height; j.width = width;
  const int x0 = (int)std::nearbyint((double)box[0]);
  const int y0 = (int)std::nearbyint((double)box[1]);
  const int x1 = (int)std::nearbyint((double)box[2]);
  const int y1 = (int)std::nearbyint((double)box[3]);
  j.sx0 = x0; j.sy0 = y0; j.cw = x1 - x0; j.ch = y1 - y0;
  if (j.cw <= 0 || j.ch <= 0) return fail(h, OAKE_ERR_INVALID, "empty crop box");
  if (squash) {
    j.rw = j.rh = out_size;
    j.cx = j.cy = 0;
    return OAKE_OK;
  }
  // torchvision Resize(int) on a PIL image, then CenterCrop
  if ((j.cw <= j.ch && j.cw == out_size) || (j.ch <= j.cw && j.ch == out_size)) {
    j.rw = j.cw; j.rh = j.ch;
  } else if (j.cw < j.ch) {
    j.rw = out_size; j.rh = (int)((double)((long)out_size * j.ch) / (double)j.cw);
  } else {
    j.rh = out_size; j.rw = (int)((double)((long)out_size * j.cw) / (double)j.ch);
  }
  j.cy = (int)std::nearbyint((j.rh - out_size) / 2.0);
  j.cx = (int)std::nearbyint((j.rw - out_size) / 2.0);
  return OAKE_OK;
}

// Tile origins along one axis [REF oadp/oake/blocks.py:40-52]: nothing below r, [0] at r, else
// n = ceil((length - r) / s) steps of near-equal integer size, the first `rem` steps one pixel longer.
void partition_axis(int length, int r, int s, std::vector<int>& out) {
  out.clear();
  if (length < r) return;
  out.push_back(0);
  if (length == r) return;
  const int n = (length - r - 1) / s + 1;
  const int q = (length - r) / n, rem = (length - r) % n;
  for (int i = 0; i < n; ++i) out.push_back(out.back() + q + (i < rem ? 1 : 0));
}

}  // namespace

extern "C" {

// How a call's n crops are cut into passes of <= cfg.max_batch crops.  Every pass runs the same kernels on nb * L token
// rows, and what a pass costs is a matter of tile counts against the chip: the GEMMs walk ceil(rows / 160 or 320) x
// ceil(N / 256) tiles in rounds of one per CU (gemm.hip: the 320-row kernel where 2 x its rounds <= the 160-row kernel's;
// a 320-row tile measured at 1.78 of a 160-row one), the fused ln_1 + in_proj + attention kernel one tile per head and group
// of `per_tile` images.  Candidates: passes at the cap with a shorter last one, and k, k + 1, k + 2 EQUAL passes (k = the
// fewest that fit) — a short last pass can run the GEMMs on a fraction of the chip, and equal passes can leave every pass
// with a nearly empty last round: 1728 crops of 50 tokens under 512 go as 3 x 512 + 192 (whole rounds of every kernel),
// not 4 x 432 (c_proj / out_proj on 80 % of the CUs, the attention kernel's sixth round at 6 %: 12 % more by this count,
// measured on ONE lane +6 %, profiles/r06/planner/; two lanes fill each other's empty rounds: +0.4 %).  The cheapest wins;
// ties, and wins below the model's resolution, keep the fewest equal passes.  Cost unit: one K-tile-length of a 160-row
// GEMM tile (x K); constant factors common to every candidate are left out.
static int plan_pass_size_core(int cap, int n, int L, int per_tile, int width, int mlp_dim, int heads, int ncu) {
  if (n <= cap || cap <= 1) return n > 0 ? std::min(n, std::max(cap, 1)) : 1;
  if (ncu <= 0) ncu = 256;
  if (per_tile < 1) per_tile = 1;
  const double C = width, F = mlp_dim;
  auto rounds = [&](long rows_per_tile, long rows, long N) {
    const long tiles = (rows + rows_per_tile - 1) / rows_per_tile * ((N + 255) / 256);
    return (double)((tiles + ncu - 1) / ncu);
  };
  auto gemm = [&](long rows, long N, double K) {
    const double r160 = rounds(160, rows, N), r320 = rounds(320, rows, N);
    return K * (2 * r320 <= r160 ? 1.78 * r320 : r160);
  };
  auto pass = [&](int nb) {
    const long rows = (long)nb * L;
    const long attn_tiles = (long)((nb + per_tile - 1) / per_tile) * heads;
    return gemm(rows, (long)F, C) + gemm(rows, (long)C, F) + gemm(rows, (long)C, C) +
           1.3 * C * (double)((attn_tiles + ncu - 1) / ncu);
  };
  auto total = [&](int per) {
    double t = 0;
    for (int b0 = 0; b0 < n; b0 += per) t += pass(std::min(per, n - b0));
    return t;
  };
  const int k0 = (n + cap - 1) / cap;
  int best = (n + k0 - 1) / k0;
  double best_cost = total(best);
  const int cands[3] = {(n + k0) / (k0 + 1), (n + k0 + 1) / (k0 + 2), cap};
  for (int per : cands) {
    if (per < 1 || per > cap) continue;
    const double t = total(per);
    if (t < best_cost * 0.99) {  // (a candidate has to win by more than the model's resolution)
      best = per;
      best_cost = t;
    }
  }
  return best;
}

static int plan_pass_size(const oake_handle* h, int n, int L, int per_tile) {
  const oake_config& c = h->cfg;
  int ncu = 0;
  if (n > c.max_batch &&
      hipDeviceGetAttribute(&ncu, hipDeviceAttributeMultiprocessorCount, h->device) != hipSuccess)
    ncu = 0;
  if (h->opts.cu_count > 0 && (ncu <= 0 || h->opts.cu_count < ncu)) ncu = h->opts.cu_count;
  return plan_pass_size_core(c.max_batch, n, L, per_tile, c.width, c.mlp_dim, c.heads, ncu);
}

// (host arithmetic only — tests/test_abi.py runs it without a GPU)
int oake_debug_plan_pass(int cap, int n, int tokens, int images_per_attention_tile, int width, int mlp_dim, int heads,
                         int compute_units) {
  return plan_pass_size_core(cap, n, tokens, images_per_attention_tile, width, mlp_dim, heads, compute_units);
}

int oake_encode_image(oake_handle* h, const void* d_images, int in_dtype, int n, void* d_out,
                      int out_dtype, int normalize, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (h->text) return fail(h, OAKE_ERR_STATE, "text handle: use oake_encode_text");
  if (n < 0) return fail(h, OAKE_ERR_INVALID, "negative batch");
  if (n == 0) return OAKE_OK;
  if (!d_images || !d_out) return fail(h, OAKE_ERR_INVALID, "null device pointer");
  if (in_dtype != OAKE_F32 && in_dtype != OAKE_F16 && in_dtype != OAKE_BF16)
    return fail(h, OAKE_ERR_INVALID, "in_dtype must be F32, F16 or BF16");
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  int rc = check_ready(h);
  if (rc) return rc;
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const oake_config& c = h->cfg;
  const int C = c.width, L = h->tokens;
  const size_t img_bytes = (size_t)3 * c.image_size * c.image_size * dtype_size(in_dtype);
  const size_t out_bytes = (size_t)c.embed_dim * dtype_size(out_dtype);

  // the pass size: plan_pass_size() — a crop's result depends on its pass only through the tile shapes the small
  // last-layer GEMMs pick for the pass's row count (rounding: <= 3e-4 on the unit-norm output, tests/test_encoder_gpu.py)
  const int per_pass = plan_pass_size(h, n, L, L <= 50 ? 4 : 1);
  for (int b0 = 0; b0 < n; b0 += per_pass) {
    const int nb = std::min(per_pass, n - b0);
    const int T = nb * L;
    const char* imgs = reinterpret_cast<const char*>(d_images) + (size_t)b0 * img_bytes;
    char* outp = reinterpret_cast<char*>(d_out) + (size_t)b0 * out_bytes;
    if ((rc = patch_embed(h, s, imgs, in_dtype, nb))) return rc;
    // Only the CLS row of the last block reaches ln_post (VisionTransformer.forward: x[:, 0, :]), so of
    // that block only its K / V projections are needed for all tokens; the query, the attention
    // output, out_proj and the MLP are computed for the CLS rows alone — the same dead-row elimination
    // as the objects stream's, through the same code: the CLS rows are copied
    // to rows T .. T+nb and attend over the patch rows + themselves (object_attention with a zero mask).
    // Identical results row for row; 6.7 % fewer FLOPs per image at 12 layers.
    const bool cls_last = h->cls_last && L >= 2 && L <= 1024;
    const size_t xs = h->xdt == DT_F32 ? 4 : 2;
    char* yrows = reinterpret_cast<char*>(h->x) + (size_t)T * C * xs;
    for (int l = 0; l < c.layers; ++l) {
      const LayerW& w = h->layers[l];
      if (l + 1 < c.layers || !cls_last) {
        if (fuses_qkv_attn(h, nb)) {
          if ((rc = main_qkv_attn(h, s, w, nb))) return rc;
          continue;
        }
        if ((rc = main_in_proj(h, s, w, T, false))) return rc;
        if ((rc = main_block_tail(h, s, w, nb))) return rc;
        continue;
      }
      RUN(h, s, "copy_cls", 0.0, 2.0 * nb * C * xs,
          hipMemcpy2DAsync(yrows, (size_t)C * xs, h->x, (size_t)L * C * xs, (size_t)C * xs, nb,
                           hipMemcpyDeviceToDevice, s));
      if ((rc = in_proj_rows(h, s, w, 0, T, true, "gemm_kv"))) return rc;
      const bool fused = h->stat_fused;
      h->stat_fused = false;  // (the small kernels take (rstd, -mean rstd) from a rowstat pass)
      rc = in_proj_rows(h, s, w, T, nb, false, "gemm_qkv_cls");
      if (rc == OAKE_OK) {
        const char* qkv_y = reinterpret_cast<const char*>(h->qkv) + (size_t)T * 3 * C * 2;
        char* att_y = reinterpret_cast<char*>(h->att) + (size_t)T * C * 2;
        RUNK(h, s, "cls_attention", 4.0 * nb * c.heads * (double)L * 64, 0.0,
             launch_object_attention(h->dt16, h->qkv, qkv_y, h->zero_mask, DT_F16, att_y, nb, L, c.heads, s, &h->opts));
        rc = mlp_rows(h, s, w, T, nb, "_cls");
      }
      h->stat_fused = fused;
      if (rc) return rc;
    }
    if (cls_last) {
      if ((rc = head(h, s, yrows, h->xdt, (long)C, outp, out_dtype, normalize, nb))) return rc;
    } else {
      if ((rc = head(h, s, h->x, h->xdt, (long)L * C, outp, out_dtype, normalize, nb))) return rc;
    }
  }
  return OAKE_OK;
}

int oake_encode_text(oake_handle* h, const int32_t* d_tokens, int n, int length, void* d_out,
                     int out_dtype, int normalize, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (!h->text) return fail(h, OAKE_ERR_STATE, "not a text handle (oake_text_create)");
  if (n < 0) return fail(h, OAKE_ERR_INVALID, "negative batch");
  if (n == 0) return OAKE_OK;
  if (!d_tokens || !d_out) return fail(h, OAKE_ERR_INVALID, "null device pointer");
  if (length <= 0 || length > h->tokens) return fail(h, OAKE_ERR_INVALID, "length must be in 1..context");
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  int rc = check_ready(h);
  if (rc) return rc;
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const oake_config& c = h->cfg;
  const int C = c.width, L = length;
  const size_t out_bytes = (size_t)c.embed_dim * dtype_size(out_dtype);
  // the workspace holds max_batch sequences of the full context; shorter sequences pack more per pass
  // ... but never more than the head buffers (gather_eot -> ln_final -> projection -> normalise) hold
  const int per_pass = (int)std::min<long>(std::min<long>(((long)c.max_batch * h->tokens) / L, h->head_rows),
                                           0x7fffffffL / (3L * C * L));
  for (int b0 = 0; b0 < n; b0 += per_pass) {
    const int nb = std::min(per_pass, n - b0);
    const int T = nb * L;
    const int32_t* toks = d_tokens + (size_t)b0 * L;
    char* outp = reinterpret_cast<char*>(d_out) + (size_t)b0 * out_bytes;
    h->cur_len = L;
    h->stat_fused = h->xdt != DT_F32 && C % 64 == 0 && C / 64 <= 16 &&
                    gemm_uses_persistent(T, C, C, &h->opts) && gemm_uses_persistent(T, C, c.mlp_dim, &h->opts) &&
                    gemm_uses_persistent(T, 3 * C, C, &h->opts) && gemm_uses_persistent(T, c.mlp_dim, C, &h->opts);
    // clip model.py encode_text: token_embedding(text) + positional_embedding[:L]
    RUN(h, s, "text_embed", 0.0, (double)T * C * 10,
        launch_text_embed(toks, h->tok_emb, h->pos, h->x, h->xdt, nb, L, C, h->vocab,
                          h->stat_fused ? h->rowpart : nullptr, s));
    h->nparts = 1;
    for (int l = 0; l < c.layers; ++l) {
      const LayerW& w = h->layers[l];
      if ((rc = main_in_proj(h, s, w, T, false))) return rc;
      if ((rc = main_block_tail(h, s, w, nb))) return rc;  // causal attention (h->text)
    }
    // x[arange(n), text.argmax(-1)] -> ln_final -> @ text_projection
    RUN(h, s, "gather_eot", 0.0, (double)nb * C * 6,
        launch_gather_eot(toks, h->x, h->xdt, h->y, nb, L, C, s));
    if ((rc = head(h, s, h->y, DT_F32, (long)C, outp, out_dtype, normalize, nb))) return rc;
  }
  return OAKE_OK;
}

int oake_encode_objects(oake_handle* h, const void* d_objects, int in_dtype, const void* d_masks,
                        int mask_dtype, int n, void* d_out, int out_dtype, int normalize,
                        void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (h->text) return fail(h, OAKE_ERR_STATE, "text handle: use oake_encode_text");
  if (n < 0) return fail(h, OAKE_ERR_INVALID, "negative batch");
  if (n == 0) return OAKE_OK;
  if (!d_objects || !d_masks || !d_out) return fail(h, OAKE_ERR_INVALID, "null device pointer");
  const bool in_padded = (in_dtype & OAKE_LAYOUT_PADDED) != 0;
  in_dtype &= ~OAKE_LAYOUT_PADDED;
  if (in_dtype != OAKE_F32 && in_dtype != OAKE_F16 && in_dtype != OAKE_BF16)
    return fail(h, OAKE_ERR_INVALID, "in_dtype must be F32, F16 or BF16");
  int ppad = 0, php = 0, pws = 0;
  if (in_padded && (!padded_geometry(h, &ppad, &php, &pws) || in_dtype != h->dt16 ||
                    reinterpret_cast<uintptr_t>(d_objects) % 16 != 0))
    return fail(h, OAKE_ERR_INVALID, "OAKE_LAYOUT_PADDED input: the handle's conv1 takes no zero-padded batch (oake_padded_layout), "
                                     "or the batch is not of the compute type / 16-byte aligned");
  if (mask_dtype != OAKE_F32 && mask_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "mask_dtype must be F32 or F16");
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  int rc = check_ready(h);
  if (rc) return rc;
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const oake_config& c = h->cfg;
  const int C = c.width, L = h->tokens;
  const size_t img_bytes = in_padded ? (size_t)3 * php * pws * 2 : (size_t)3 * c.image_size * c.image_size * dtype_size(in_dtype);
  const size_t mask_bytes = (size_t)h->p2 * dtype_size(mask_dtype);
  const size_t out_bytes = (size_t)c.embed_dim * dtype_size(out_dtype);

  // the pass size: plan_pass_size() (as oake_encode_image)
  const int per_pass = plan_pass_size(h, n, L, 1);
  for (int b0 = 0; b0 < n; b0 += per_pass) {
    const int nb = std::min(per_pass, n - b0);
    const int T = nb * L;
    const char* imgs = reinterpret_cast<const char*>(d_objects) + (size_t)b0 * img_bytes;
    const char* masks = reinterpret_cast<const char*>(d_masks) + (size_t)b0 * mask_bytes;
    char* outp = reinterpret_cast<char*>(d_out) + (size_t)b0 * out_bytes;
    if ((rc = patch_embed(h, s, imgs, in_dtype, nb, in_padded))) return rc;
    // Hooks.transformer_forward_pre (objects.py:215-221): y = x[[0]] (after ln_pre).  The object
    // tokens live as rows T .. T+nb of the SAME matrices as the patch tokens, so that every layer's
    // GEMMs carry both streams in one launch (they share the weights); only the attention differs.
    const size_t xs = h->xdt == DT_F32 ? 4 : 2;
    char* yrows = reinterpret_cast<char*>(h->x) + (size_t)T * C * xs;
    RUN(h, s, "copy_cls", 0.0, 2.0 * nb * C * xs,
        hipMemcpy2DAsync(yrows, (size_t)C * xs, h->x, (size_t)L * C * xs, (size_t)C * xs, nb,
                         hipMemcpyDeviceToDevice, s));
    if (h->stat_fused)  // ... and so do their row statistics (slot 0 of the CLS rows)
      HIP_TRY(h, hipMemcpy2DAsync(h->rowpart + (size_t)T * 32, 32 * 4, h->rowpart, (size_t)L * 32 * 4, 8, nb,
                                  hipMemcpyDeviceToDevice, s));
    const char* qkv_y = reinterpret_cast<const char*>(h->qkv) + (size_t)T * 3 * C * 2;
    char* att_y = reinterpret_cast<char*>(h->att) + (size_t)T * C * 2;
    for (int l = 0; l < c.layers; ++l) {
      const LayerW& w = h->layers[l];
      const bool last = (l == c.layers - 1);
      if (!last && fuses_qkv_attn_obj(h, nb) && w.in_wfp) {
        // ... as one kernel per layer: a tile = (crop, head), the crop's object token rides as row L of the tile
        int np = 0;
        if ((rc = ln_stats(h, s, reinterpret_cast<const char*>(h->x), 0, T + nb, 3 * C, C, &np))) return rc;
        if (np < 1) return fail(h, OAKE_ERR_STATE, "qkv_attn_obj: no row statistics");
        RUNK(h, s, "qkv_attn", 2.0 * (T + nb) * 3 * C * C + 4.0 * nb * c.heads * ((double)L * L + L) * 64, 0.0,
             launch_qkv_attn_obj(h->dt16, h->x, w.in_wfp, w.in_bfp, w.in_csp, h->rowpart, np, masks, mask_dtype, h->att,
                                 nb, L, c.heads, &h->opts, s));
        if ((rc = mlp_rows(h, s, w, 0, T + nb, ""))) return rc;
        continue;
      }
      if (!last) {
        // ln_1 + in-proj of both streams; k/v of the patch rows serve both (Appendix C #1)
        if ((rc = in_proj_rows(h, s, w, 0, T + nb, false, "gemm_qkv"))) return rc;
      } else {
        // last layer: the main stream's q is dead and its block is never run (Appendix C #2) —
        // k and v of the patch rows, then the object tokens on their own (small GEMMs, once)
        if ((rc = in_proj_rows(h, s, w, 0, T, true, "gemm_kv"))) return rc;
        const bool fused = h->stat_fused;
        h->stat_fused = false;  // (the small kernels take (rstd, -mean rstd) from a rowstat pass)
        rc = in_proj_rows(h, s, w, T, nb, false, "gemm_qkv_y");
        h->stat_fused = fused;
        if (rc) return rc;
      }
      // object-token attention (Hooks.residual_attention_block_forward_pre, objects.py:223-247): on an
      // idle wave of the main stream's attention launch when there is one, else its own kernel
      const bool fuse = !last && attention_fuses_object_token(L, &h->opts);
      if (!fuse)
        RUNK(h, s, "object_attention", 4.0 * nb * c.heads * (double)L * 64, 0.0,
            launch_object_attention(h->dt16, h->qkv, qkv_y, masks, mask_dtype, att_y, nb, L, c.heads, s, &h->opts));
      if (!last) {
        const int Lp = L;  // (algorithmic FLOPs, as main_block_tail)
        RUNK(h, s, "attention", 4.0 * nb * c.heads * (double)Lp * Lp * 64, (double)T * 4 * C * 2,
            launch_attention(h->dt16, h->qkv, h->att, nb, L, c.heads, 0, s, fuse ? qkv_y : nullptr,
                             fuse ? masks : nullptr, mask_dtype, fuse ? att_y : nullptr, &h->opts));
        if ((rc = mlp_rows(h, s, w, 0, T + nb, ""))) return rc;
      } else {
        const bool fused = h->stat_fused;
        h->stat_fused = false;
        rc = mlp_rows(h, s, w, T, nb, "_y");
        h->stat_fused = fused;
        if (rc) return rc;
      }
    }
    // Hooks.transformer_forward (objects.py:249-258): the block stack's output is y
    if ((rc = head(h, s, yrows, h->xdt, (long)C, outp, out_dtype, normalize, nb))) return rc;
  }
  return OAKE_OK;
}

int oake_crop_normalize(oake_handle* h, const uint8_t* d_image_hwc, int height, int width,
                        const int32_t* d_boxes_xyxy, int k, int out_size, const float* h_mean3,
                        const float* h_std3, void* d_out, int out_dtype, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (k < 0 || height <= 0 || width <= 0 || out_size <= 0)
    return fail(h, OAKE_ERR_INVALID, "bad crop geometry");
  if (k == 0) return OAKE_OK;
  if (!d_image_hwc || !d_boxes_xyxy || !d_out || !h_mean3 || !h_std3)
    return fail(h, OAKE_ERR_INVALID, "null pointer");
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const double bytes = (double)k * out_size * out_size * 3 * (1 + dtype_size(out_dtype));
  RUN(h, s, "crop_normalize", 0.0, bytes,
      launch_crop_normalize(d_image_hwc, height, width, d_boxes_xyxy, k, out_size, h_mean3, h_std3,
                            d_out, out_dtype, s));
  return OAKE_OK;
}

int oake_crop_resize_normalize(oake_handle* h, const uint8_t* d_image_hwc, int height, int width,
                               const float* h_boxes_xyxy, int k, int out_size, int squash,
                               const float* h_mean3, const float* h_std3, void* d_out, int out_dtype,
                               void* stream) {
  const int counts[1] = {k};
  const uint8_t* const imgs[1] = {d_image_hwc};
  return oake_crop_resize_normalize_batch(h, 1, imgs, &height, &width, h_boxes_xyxy, counts, out_size, squash,
                                          h_mean3, h_std3, d_out, out_dtype, stream);
}

int oake_crop_resize_normalize_batch(oake_handle* h, int n_images, const uint8_t* const* d_images,
                                     const int* heights, const int* widths, const float* h_boxes_xyxy,
                                     const int* counts, int out_size, int squash, const float* h_mean3,
                                     const float* h_std3, void* d_out, int out_dtype, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (n_images < 0 || out_size <= 0) return fail(h, OAKE_ERR_INVALID, "bad crop geometry");
  if (n_images == 0) return OAKE_OK;
  if (!d_images || !heights || !widths || !counts || !h_mean3 || !h_std3)
    return fail(h, OAKE_ERR_INVALID, "null pointer");
  const bool out_padded = (out_dtype & OAKE_LAYOUT_PADDED) != 0;
  out_dtype &= ~OAKE_LAYOUT_PADDED;
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  int ppad = 0, php = 0, pws = 0;
  if (out_padded && (!padded_geometry(h, &ppad, &php, &pws) || out_dtype != h->dt16 || out_dtype != OAKE_F16 ||
                     out_size != h->cfg.image_size || reinterpret_cast<uintptr_t>(d_out) % 16 != 0))
    return fail(h, OAKE_ERR_INVALID, "OAKE_LAYOUT_PADDED output: f16 crops of the handle's image size into the zero-padded batch "
                                     "of a handle whose conv1 pads (oake_padded_layout)");
  size_t total = 0;
  for (int i = 0; i < n_images; ++i) {
    if (counts[i] < 0) return fail(h, OAKE_ERR_INVALID, "negative box count");
    if (counts[i] > 0 && (!d_images[i] || heights[i] <= 0 || widths[i] <= 0))
      return fail(h, OAKE_ERR_INVALID, "bad crop geometry");
    total += (size_t)counts[i];
  }
  if (total == 0) return OAKE_OK;
  if (!h_boxes_xyxy || !d_out) return fail(h, OAKE_ERR_INVALID, "null pointer");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // the crops of ALL images as one job list: three launches per call, whatever the number of images
  std::vector<ResampleJob> jobs(total);
  size_t k = 0;
  for (int i = 0; i < n_images; ++i)
    for (int c = 0; c < counts[i]; ++c, ++k) {
      const int rc = fill_crop_job(h, jobs[k], d_images[i], heights[i], widths[i], h_boxes_xyxy + 4 * k, out_size,
                                   squash);
      if (rc != OAKE_OK) return rc;
      jobs[k].out_row = (long)k;
    }
  return run_resample(h, s, jobs, out_size, h_mean3, h_std3, d_out, out_dtype, out_padded ? ppad : 0, out_padded ? php : 0,
                      out_padded ? pws : 0);
}

int oake_padded_layout(const oake_handle* h, int* padding, int* rows, int* row_stride) {
  if (!h || !padding || !rows || !row_stride) return OAKE_ERR_INVALID;
  int p = 0, hp = 0, ws = 0;
  if (!padded_geometry(h, &p, &hp, &ws)) return OAKE_ERR_UNSUPPORTED;
  *padding = p; *rows = hp; *row_stride = ws;
  return OAKE_OK;
}

int oake_resize_u8(oake_handle* h, const uint8_t* d_src_hwc, int sh, int sw, uint8_t* d_dst_hwc,
                   int dh, int dw, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (sh <= 0 || sw <= 0 || dh <= 0 || dw <= 0 || !d_src_hwc || !d_dst_hwc)
    return fail(h, OAKE_ERR_INVALID, "bad resize arguments");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  std::vector<ResampleJob> jobs(1);
  ResampleJob& j = jobs[0];
  j = ResampleJob{};
  j.img = d_src_hwc; j.height = sh; j.width = sw;
  j.sx0 = j.sy0 = 0; j.cw = sw; j.ch = sh; j.rw = dw; j.rh = dh; j.cx = j.cy = 0;
  j.u8_out = d_dst_hwc;
  const float z[3] = {0.f, 0.f, 0.f}, o[3] = {1.f, 1.f, 1.f};
  return run_resample(h, s, jobs, 0, z, o, nullptr, OAKE_U8);
}

int oake_blocks_count(int width, int height, int block_size, int max_stride, double rescale) {
  if (width <= 0 || height <= 0 || block_size <= 0 || max_stride <= 0 || !(rescale > 1.0)) return -1;
  std::vector<int> px, py;
  long n = 1;  // block 0: the whole image
  for (int w = width, hh = height;;) {
    partition_axis(w, block_size, max_stride, px);
    partition_axis(hh, block_size, max_stride, py);
    if (px.empty() || py.empty()) break;
    n += (long)px.size() * (long)py.size();
    w = (int)((double)w / rescale);
    hh = (int)((double)hh / rescale);
  }
  return n > 0x7fffffffL ? -1 : (int)n;
}

int oake_blocks_batch(oake_handle* h, int n_images, const uint8_t* const* d_images, const int* heights,
                      const int* widths, int block_size, int max_stride, double rescale,
                      const float* h_mean3, const float* h_std3, void* d_out, int out_dtype, int* counts_out,
                      void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (n_images < 0 || block_size <= 0 || block_size % 8 != 0 || max_stride <= 0 || !(rescale > 1.0))
    return fail(h, OAKE_ERR_INVALID, "bad block geometry (block_size: positive multiple of 8; rescale > 1)");
  if (n_images == 0) return OAKE_OK;
  if (!d_images || !heights || !widths || !h_mean3 || !h_std3 || !d_out)
    return fail(h, OAKE_ERR_INVALID, "null pointer");
  if (out_dtype != OAKE_F32 && out_dtype != OAKE_F16)
    return fail(h, OAKE_ERR_INVALID, "out_dtype must be F32 or F16");
  if (reinterpret_cast<uintptr_t>(d_out) % 16 != 0)  // the crop kernels store 16-byte vectors
    return fail(h, OAKE_ERR_INVALID, "d_out must be 16-byte aligned");
  for (int i = 0; i < n_images; ++i)
    if (!d_images[i] || heights[i] <= 0 || widths[i] <= 0) return fail(h, OAKE_ERR_INVALID, "bad image");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int r = block_size;
  const int odt = out_dtype == OAKE_F32 ? DT_F32 : DT_F16;

  // ---- index math of the whole flush: the reference's _partitions walk (blocks.py:54-77) ----
  struct Level {
    int w, h;
    std::vector<int> px, py;
    size_t pyr_off;   // levels >= 1: byte offset of the level image in the pyramid arena
    size_t first_row; // output row of the level's first crop
  };
  std::vector<std::vector<Level>> levels(n_images);
  std::vector<size_t> block0_row(n_images);
  size_t rows = 0, pyr_bytes = 0, max_levels = 0;
  for (int i = 0; i < n_images; ++i) {
    block0_row[i] = rows++;
    int w = widths[i], hh = heights[i];
    for (;;) {
      Level lv;
      lv.w = w; lv.h = hh; lv.pyr_off = 0; lv.first_row = rows;
      partition_axis(w, r, max_stride, lv.px);
      partition_axis(hh, r, max_stride, lv.py);
      if (lv.px.empty() || lv.py.empty()) break;  // "halt when either side is below the block size"
      rows += lv.px.size() * lv.py.size();
      if (!levels[i].empty()) {
        lv.pyr_off = pyr_bytes;
        pyr_bytes += (((size_t)w * hh * 3) + 255) & ~(size_t)255;
      }
      levels[i].push_back(std::move(lv));
      w = (int)((double)w / rescale);   // Python int(w / rescale): float division, truncation
      hh = (int)((double)hh / rescale);
    }
    if (counts_out) counts_out[i] = (int)(rows - block0_row[i]);
    max_levels = std::max(max_levels, levels[i].size());
  }
  int rc;
  if ((rc = grow(h, s, &h->pyr, &h->pyr_cap, pyr_bytes))) return rc;

  // ---- block 0 of every image = preprocess(whole image): Resize(r, BICUBIC) + CenterCrop(r) ----
  std::vector<ResampleJob> jobs(n_images);
  for (int i = 0; i < n_images; ++i) {
    const float box[4] = {0.f, 0.f, (float)widths[i], (float)heights[i]};
    if ((rc = fill_crop_job(h, jobs[i], d_images[i], heights[i], widths[i], box, r, 0))) return rc;
    jobs[i].out_row = (long)block0_row[i];
  }
  if ((rc = run_resample(h, s, jobs, r, h_mean3, h_std3, d_out, odt))) return rc;

  // ---- level by level: the exact-size crops of ALL images' level L in one launch, then the resizes
  //      that make level L + 1 of all images (skipped where the next level has no tiles) ----
  std::vector<CropJob> cjobs;
  for (size_t L = 0; L < max_levels; ++L) {
    cjobs.clear();
    jobs.clear();
    for (int i = 0; i < n_images; ++i) {
      if (L >= levels[i].size()) continue;
      const Level& lv = levels[i][L];
      const uint8_t* src = L == 0 ? d_images[i] : h->pyr + lv.pyr_off;
      long row = (long)lv.first_row;
      for (int x : lv.px)  // itertools.product(partition(w), partition(h)): x outer, y inner
        for (int y : lv.py) cjobs.push_back(CropJob{src, lv.h, lv.w, x, y, row++});
      if (L + 1 < levels[i].size()) {
        const Level& nx = levels[i][L + 1];
        ResampleJob j{};
        j.img = src; j.height = lv.h; j.width = lv.w;
        j.cw = lv.w; j.ch = lv.h; j.rw = nx.w; j.rh = nx.h;
        j.u8_out = h->pyr + nx.pyr_off;
        jobs.push_back(j);
      }
    }
    if (!cjobs.empty()) {
      if ((rc = grow(h, s, &h->crop_jobs, &h->crop_jobs_cap, cjobs.size() * sizeof(CropJob)))) return rc;
      if ((rc = upload_async(h, s, cjobs.data(), cjobs.size() * sizeof(CropJob), h->crop_jobs))) return rc;
      RUN(h, s, "crop_normalize", 0.0, (double)cjobs.size() * r * r * 3 * (1 + (odt == DT_F32 ? 4 : 2)),
          launch_crop_normalize_jobs(h->crop_jobs, (int)cjobs.size(), r, h_mean3, h_std3, d_out, odt, s));
    }
    if (!jobs.empty()) {
      const float z[3] = {0.f, 0.f, 0.f}, o[3] = {1.f, 1.f, 1.f};
      if ((rc = run_resample(h, s, jobs, 0, z, o, nullptr, DT_U8))) return rc;
    }
  }
  return OAKE_OK;
}

int oake_jpeg_info(const uint8_t* h_data, size_t nbytes, int* height, int* width, int* components) {
  if (!h_data) return OAKE_ERR_INVALID;
  JpegFrame f;
  const int rc = jpeg_read_frame(h_data, nbytes, &f, nullptr);
  if (rc == JPEG_UNSUPPORTED) return OAKE_ERR_UNSUPPORTED;
  if (rc != JPEG_OK) return OAKE_ERR_INVALID;
  if (height) *height = f.height;
  if (width) *width = f.width;
  if (components) *components = f.ncomp;
  return OAKE_OK;
}

int oake_jpeg_info_batch(int n, const uint8_t* const* h_datas, const size_t* nbytes, int* heights,
                         int* widths, int* status) {
  if (n < 0 || (n > 0 && (!h_datas || !nbytes || !heights || !widths || !status))) return OAKE_ERR_INVALID;
  for (int i = 0; i < n; ++i) {
    heights[i] = widths[i] = 0;
    status[i] = oake_jpeg_info(h_datas[i], nbytes[i], &heights[i], &widths[i], nullptr);
  }
  return OAKE_OK;
}

int oake_jpeg_entropy_decode(const uint8_t* h_data, size_t nbytes, int16_t* h_coefs, size_t capacity,
                          size_t* total) {
  if (!h_data) return OAKE_ERR_INVALID;
  JpegFrame f;
  int rc = jpeg_read_frame(h_data, nbytes, &f, nullptr);
  if (rc == JPEG_UNSUPPORTED) return OAKE_ERR_UNSUPPORTED;
  if (rc != JPEG_OK) return OAKE_ERR_INVALID;
  if (total) *total = (size_t)f.total_coefs;
  if (!h_coefs) return OAKE_OK;
  if (capacity < (size_t)f.total_coefs) return OAKE_ERR_INVALID;
  rc = jpeg_decode_coefs(h_data, nbytes, f, h_coefs, nullptr);
  return rc == JPEG_OK ? OAKE_OK : (rc == JPEG_UNSUPPORTED ? OAKE_ERR_UNSUPPORTED : OAKE_ERR_INVALID);
}

namespace {

// frame walk + scratch sizing shared by the two decode entry points; leaves jp_host writable
int jpeg_prepare(oake_handle* h, hipStream_t s, const uint8_t* h_data, size_t nbytes, size_t out_capacity,
                 JpegFrame* f, int* height, int* width) {
  std::string err;
  int rc = jpeg_read_frame(h_data, nbytes, f, &err);
  if (rc != JPEG_OK)
    return fail(h, rc == JPEG_UNSUPPORTED ? OAKE_ERR_UNSUPPORTED : OAKE_ERR_INVALID, "jpeg: " + err);
  if (height) *height = f->height;
  if (width) *width = f->width;
  if ((size_t)f->height * f->width * 3 > out_capacity)
    return fail(h, OAKE_ERR_INVALID, "jpeg: output buffer too small");
  const size_t cbytes = (size_t)f->total_coefs * sizeof(int16_t);
  if (!h->jp_copied) HIP_TRY(h, hipEventCreateWithFlags(&h->jp_copied, hipEventDisableTiming));
  if (cbytes > h->jp_host_cap) {
    HIP_TRY(h, hipEventSynchronize(h->jp_copied));
    if (h->jp_host) HIP_TRY(h, hipHostFree(h->jp_host));
    h->jp_host = nullptr;
    h->jp_host_cap = 0;
    const size_t cap = cbytes + cbytes / 4 + 4096;
    HIP_TRY(h, hipHostMalloc(reinterpret_cast<void**>(&h->jp_host), cap, hipHostMallocDefault));
    h->jp_host_cap = cap;
  }
  if ((rc = grow(h, s, &h->jp_coefs, &h->jp_coefs_cap, cbytes))) return rc;
  if ((rc = grow(h, s, &h->jp_planes, &h->jp_planes_cap, (size_t)f->total_plane_bytes))) return rc;
  // the previous image's coefficients must have left the pinned buffer before it is rewritten
  HIP_TRY(h, hipEventSynchronize(h->jp_copied));
  return OAKE_OK;
}

int jpeg_upload_and_reconstruct(oake_handle* h, hipStream_t s, const JpegFrame& f, uint8_t* d_out_hwc) {
  const size_t cbytes = (size_t)f.total_coefs * sizeof(int16_t);
  HIP_TRY(h, hipMemcpyAsync(h->jp_coefs, h->jp_host, cbytes, hipMemcpyHostToDevice, s));
  HIP_TRY(h, hipEventRecord(h->jp_copied, s));
  RUN(h, s, "jpeg_reconstruct", 0.0, (double)cbytes + 2.0 * f.total_plane_bytes + 3.0 * f.height * f.width,
      launch_jpeg_reconstruct(f, h->jp_coefs, h->jp_planes, d_out_hwc, s));
  return OAKE_OK;
}

}  // namespace

int oake_decode_jpeg(oake_handle* h, const uint8_t* h_data, size_t nbytes, uint8_t* d_out_hwc,
                     size_t out_capacity, int* height, int* width, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (!h_data || !d_out_hwc) return fail(h, OAKE_ERR_INVALID, "null pointer");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  JpegFrame f;
  int rc = jpeg_prepare(h, s, h_data, nbytes, out_capacity, &f, height, width);
  if (rc) return rc;
  std::string err;
  rc = jpeg_decode_coefs(h_data, nbytes, f, h->jp_host, &err);
  if (rc != JPEG_OK)
    return fail(h, rc == JPEG_UNSUPPORTED ? OAKE_ERR_UNSUPPORTED : OAKE_ERR_INVALID, "jpeg: " + err);
  return jpeg_upload_and_reconstruct(h, s, f, d_out_hwc);
}

int oake_decode_jpeg_batch(oake_handle* h, int n, const uint8_t* const* h_datas, const size_t* nbytes,
                           uint8_t* const* d_outs, const size_t* capacities, int* heights, int* widths,
                           int* status, int threads, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (n < 0) return fail(h, OAKE_ERR_INVALID, "negative batch");
  if (n == 0) return OAKE_OK;
  if (!h_datas || !nbytes || !d_outs || !capacities || !status)
    return fail(h, OAKE_ERR_INVALID, "null pointer");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // 1. headers (serial, microseconds each): which images we take, and how much scratch they need
  std::vector<JpegFrame> frames(n);
  std::vector<size_t> coff(n, 0), poff(n, 0);
  size_t ctotal = 0, ptotal = 0;
  for (int i = 0; i < n; ++i) {
    const int rc = (h_datas[i] && d_outs[i]) ? jpeg_read_frame(h_datas[i], nbytes[i], &frames[i], nullptr)
                                              : JPEG_INVALID;
    status[i] = rc == JPEG_OK ? OAKE_OK : (rc == JPEG_UNSUPPORTED ? OAKE_ERR_UNSUPPORTED : OAKE_ERR_INVALID);
    if (status[i] == OAKE_OK && (size_t)frames[i].height * frames[i].width * 3 > capacities[i])
      status[i] = OAKE_ERR_INVALID;
    if (heights) heights[i] = rc == JPEG_OK ? frames[i].height : 0;
    if (widths) widths[i] = rc == JPEG_OK ? frames[i].width : 0;
    if (status[i] != OAKE_OK) continue;
    coff[i] = ctotal;
    poff[i] = ptotal;
    ctotal += (size_t)frames[i].total_coefs;
    ptotal += ((size_t)frames[i].total_plane_bytes + 15) & ~(size_t)15;
  }
  if (ctotal == 0) return OAKE_OK;
  const size_t cbytes = ctotal * sizeof(int16_t);
  if (!h->jp_copied) HIP_TRY(h, hipEventCreateWithFlags(&h->jp_copied, hipEventDisableTiming));
  HIP_TRY(h, hipEventSynchronize(h->jp_copied));  // the pinned buffer's previous contents are on the device
  if (cbytes > h->jp_host_cap) {
    if (h->jp_host) HIP_TRY(h, hipHostFree(h->jp_host));
    h->jp_host = nullptr;
    h->jp_host_cap = 0;
    const size_t cap = cbytes + cbytes / 4 + 4096;
    HIP_TRY(h, hipHostMalloc(reinterpret_cast<void**>(&h->jp_host), cap, hipHostMallocDefault));
    h->jp_host_cap = cap;
  }
  int rc;
  if ((rc = grow(h, s, &h->jp_coefs, &h->jp_coefs_cap, cbytes))) return rc;
  if ((rc = grow(h, s, &h->jp_planes, &h->jp_planes_cap, ptotal))) return rc;
  // 2. the Huffman passes: independent serial bit streams, one image per task on `threads` host threads
  {
    std::atomic<int> next(0);
    auto work = [&]() {
      for (int i = next.fetch_add(1); i < n; i = next.fetch_add(1)) {
        if (status[i] != OAKE_OK) continue;
        const int r2 = jpeg_decode_coefs(h_datas[i], nbytes[i], frames[i], h->jp_host + coff[i], nullptr);
        if (r2 != JPEG_OK) status[i] = r2 == JPEG_UNSUPPORTED ? OAKE_ERR_UNSUPPORTED : OAKE_ERR_INVALID;
      }
    };
    const int nt = std::max(1, std::min(threads, n));
    std::vector<std::thread> pool;
    for (int t = 1; t < nt; ++t) pool.emplace_back(work);
    work();
    for (auto& t : pool) t.join();
  }
  // 3. one upload, then IDCT + upsampling + colour conversion per image
  HIP_TRY(h, hipMemcpyAsync(h->jp_coefs, h->jp_host, cbytes, hipMemcpyHostToDevice, s));
  HIP_TRY(h, hipEventRecord(h->jp_copied, s));
  for (int i = 0; i < n; ++i) {
    if (status[i] != OAKE_OK) continue;
    const JpegFrame& f = frames[i];
    RUN(h, s, "jpeg_reconstruct", 0.0,
        (double)f.total_coefs * 2 + 2.0 * f.total_plane_bytes + 3.0 * f.height * f.width,
        launch_jpeg_reconstruct(f, h->jp_coefs + coff[i], h->jp_planes + poff[i], d_outs[i], s));
  }
  return OAKE_OK;
}

int oake_jpeg_reconstruct(oake_handle* h, const uint8_t* h_data, size_t nbytes, const int16_t* h_coefs,
                          size_t ncoefs, uint8_t* d_out_hwc, size_t out_capacity, int* height,
                          int* width, void* stream) {
  if (!h) return OAKE_ERR_INVALID;
  if (!h_data || !h_coefs || !d_out_hwc) return fail(h, OAKE_ERR_INVALID, "null pointer");
  HIP_TRY(h, hipSetDevice(h->device));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  JpegFrame f;
  int rc = jpeg_prepare(h, s, h_data, nbytes, out_capacity, &f, height, width);
  if (rc) return rc;
  if (ncoefs != (size_t)f.total_coefs)
    return fail(h, OAKE_ERR_INVALID, "jpeg: coefficient count does not match the frame header");
  std::memcpy(h->jp_host, h_coefs, ncoefs * sizeof(int16_t));
  return jpeg_upload_and_reconstruct(h, s, f, d_out_hwc);
}

int oake_profile_enable(oake_handle* h, int enable) {
  if (!h) return OAKE_ERR_INVALID;
  if (!enable) prof_collect(h);
  h->prof = enable != 0;
  h->prof_stride = enable > 1 ? enable : 1;
  h->prof_seq = 0;
  return OAKE_OK;
}

int oake_profile_reset(oake_handle* h) {
  if (!h) return OAKE_ERR_INVALID;
  prof_collect(h);
  h->slots.clear();
  return OAKE_OK;
}

int oake_profile_read(oake_handle* h, oake_profile_entry* entries, int cap, int* count) {
  if (!h || !count) return OAKE_ERR_INVALID;
  HIP_TRY(h, hipSetDevice(h->device));
  prof_collect(h);
  const int n = (int)h->slots.size();
  *count = n;
  for (int i = 0; i < n && i < cap && entries; ++i) {
    std::memset(&entries[i], 0, sizeof(entries[i]));
    std::snprintf(entries[i].name, sizeof(entries[i].name), "%s", h->slots[i].name.c_str());
    entries[i].total_ms = h->slots[i].ms;
    entries[i].flops = h->slots[i].flops;
    entries[i].bytes = h->slots[i].bytes;
    entries[i].launches = h->slots[i].launches;
    entries[i].seen = h->slots[i].seen;
  }
  return OAKE_OK;
}

// ---- kernel-level test entry points -----------------------------------------------------------
static int dbg(hipError_t e) { return e == hipSuccess ? OAKE_OK : OAKE_ERR_HIP; }

int oake_debug_gemm(const void* d_a, const void* d_w, const float* d_bias, float* d_c, int m, int n,
                    int k, int dtype16, void* stream) {
  GemmArgs a{};
  a.A = d_a; a.W = d_w; a.bias = d_bias; a.out = d_c; a.M = m; a.N = n; a.K = k; a.ldo = n;
  a.opts = &t_debug_opts;
  return dbg(launch_gemm(dtype16, EPI_F32_BIAS, a, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_gemm16(const void* d_a, const void* d_w, const float* d_bias, void* d_c, int m, int n,
                      int k, int dtype16, int gelu, void* stream) {
  GemmArgs a{};
  a.A = d_a; a.W = d_w; a.bias = d_bias; a.out = d_c; a.M = m; a.N = n; a.K = k; a.ldo = n;
  a.opts = &t_debug_opts;
  // gelu: 0 bias, 1 bias + QuickGELU; measurement-only: 2 = no epilogue at all, 3 = pack + store only
  const int epi = gelu == 1 ? EPI_T16_GELU : gelu == 2 ? EPI_T16_NONE : gelu == 3 ? EPI_T16_RAW : EPI_T16_BIAS;
  return dbg(launch_gemm(dtype16, epi, a, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_ln_gemm16(const void* d_x, const float* d_w32, const float* d_gamma,
                         const float* d_beta, const float* d_bias, void* d_c, int m, int n, int k,
                         int dtype16, int gelu, void* stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void* wf = nullptr;
  float *cs = nullptr, *bf = nullptr, *stat = nullptr;
  hipError_t e = hipMalloc(&wf, (size_t)n * k * 2);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&cs), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bf), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&stat), ((size_t)m + 2) * 8);
  if (e == hipSuccess) e = launch_fold_ln(dtype16, d_w32, d_gamma, d_beta, d_bias, wf, cs, bf, n, k, s);
  float* part = nullptr;
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&part), (size_t)m * 32 * 4);
  if (e == hipSuccess) e = launch_rowstat(d_x, dtype16, k, stat, m, k, s);
  if (e == hipSuccess) e = launch_rowsums(d_x, dtype16, k, part, m, k, s);
  if (e == hipSuccess) {
    GemmArgs a{};
    a.A = d_x; a.W = wf; a.bias = bf; a.out = d_c; a.M = m; a.N = n; a.K = k; a.ldo = n;
    a.rowstat = stat; a.colsum = cs; a.rowpart_in = part; a.nparts = 1;
    a.opts = &t_debug_opts;
    e = launch_gemm(dtype16, gelu ? EPI_T16_GELU_LN : EPI_T16_BIAS_LN, a, s);
  }
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  (void)hipFree(wf); (void)hipFree(cs); (void)hipFree(bf); (void)hipFree(stat); (void)hipFree(part);
  return dbg(e);
}

int oake_debug_ln_qkv_attn(const void* d_x, const float* d_w32, const float* d_gamma, const float* d_beta,
                           const float* d_bias, void* d_out, int n_img, int l, int heads, int dtype16, void* d_trace,
                           int repeats, void* stream) {
#if !OAKE_LAB
  // (the three-image form lost its A/B to the four-image one — docs/history/round5.md item 11 — and lives in liboake_hip_lab.so only)
  (void)d_x; (void)d_w32; (void)d_gamma; (void)d_beta; (void)d_bias; (void)d_out; (void)n_img; (void)l; (void)heads;
  (void)dtype16; (void)d_trace; (void)repeats; (void)stream;
  return OAKE_ERR_UNSUPPORTED;
#else
  const int C = heads * 64, n = 3 * C, m = n_img * l;
  if (!d_x || !d_w32 || !d_gamma || !d_beta || !d_bias || !d_out || n_img < 1) return OAKE_ERR_INVALID;
  if (!qkv_attn_supported(l, heads, C, n_img)) return OAKE_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void *wf = nullptr, *wp = nullptr;
  float *cs = nullptr, *bf = nullptr, *csp = nullptr, *bfp = nullptr, *part = nullptr;
  hipError_t e = hipMalloc(&wf, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(&wp, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&cs), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bf), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&csp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bfp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&part), (size_t)m * 32 * 4);
  if (e == hipSuccess) e = launch_fold_ln(dtype16, d_w32, d_gamma, d_beta, d_bias, wf, cs, bf, n, C, s);
  if (e == hipSuccess) e = launch_rowsums(d_x, dtype16, C, part, m, C, s);
  if (e == hipSuccess) e = launch_permute_qkv(dtype16, wf, bf, cs, wp, bfp, csp, C, s);
  for (int i = 0; i < (repeats < 1 ? 1 : repeats) && e == hipSuccess; ++i)
    e = launch_qkv_attn(dtype16, d_x, wp, bfp, csp, part, 1, d_out, n_img, l, heads, &t_debug_opts, s,
                        reinterpret_cast<unsigned long long*>(d_trace));
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  (void)hipFree(wf); (void)hipFree(wp); (void)hipFree(cs); (void)hipFree(bf); (void)hipFree(csp); (void)hipFree(bfp);
  (void)hipFree(part);
  return dbg(e);
#endif
}

int oake_debug_ln_qkv_attn_quad(const void* d_x, const float* d_w32, const float* d_gamma, const float* d_beta,
                                const float* d_bias, void* d_out, int n_img, int l, int heads, int dtype16, void* d_trace,
                                int repeats, void* stream) {
  const int C = heads * 64, n = 3 * C, m = n_img * l;
  if (!d_x || !d_w32 || !d_gamma || !d_beta || !d_bias || !d_out || n_img < 1) return OAKE_ERR_INVALID;
  if (!qkv_attn_quad_supported(l, heads, C, n_img)) return OAKE_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void *wf = nullptr, *wp = nullptr;
  float *cs = nullptr, *bf = nullptr, *csp = nullptr, *bfp = nullptr, *part = nullptr;
  hipError_t e = hipMalloc(&wf, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(&wp, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&cs), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bf), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&csp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bfp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&part), (size_t)m * 32 * 4);
  if (e == hipSuccess) e = launch_fold_ln(dtype16, d_w32, d_gamma, d_beta, d_bias, wf, cs, bf, n, C, s);
  if (e == hipSuccess) e = launch_rowsums(d_x, dtype16, C, part, m, C, s);
  if (e == hipSuccess) e = launch_permute_qkv_obj(wf, bf, cs, wp, bfp, csp, C, s);
  for (int i = 0; i < (repeats < 1 ? 1 : repeats) && e == hipSuccess; ++i)
    e = launch_qkv_attn_quad(dtype16, d_x, wp, bfp, csp, part, 1, d_out, n_img, l, heads, &t_debug_opts, s,
                             reinterpret_cast<unsigned long long*>(d_trace));
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  (void)hipFree(wf); (void)hipFree(wp); (void)hipFree(cs); (void)hipFree(bf); (void)hipFree(csp); (void)hipFree(bfp);
  (void)hipFree(part);
  return dbg(e);
}

int oake_debug_ln_qkv_attn_obj(const void* d_x, const float* d_w32, const float* d_gamma, const float* d_beta,
                               const float* d_bias, const void* d_mask, int mask_dtype, void* d_out, int n_img, int l,
                               int heads, int dtype16, void* d_trace, int repeats, void* stream) {
  const int C = heads * 64, n = 3 * C, m = n_img * l + n_img;
  if (!d_x || !d_w32 || !d_gamma || !d_beta || !d_bias || !d_mask || !d_out || n_img < 1) return OAKE_ERR_INVALID;
  if (!qkv_attn_obj_supported(l, heads, C, n_img)) return OAKE_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void *wf = nullptr, *wp = nullptr;
  float *cs = nullptr, *bf = nullptr, *csp = nullptr, *bfp = nullptr, *part = nullptr;
  hipError_t e = hipMalloc(&wf, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(&wp, (size_t)n * C * 2);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&cs), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bf), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&csp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&bfp), (size_t)n * 4);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&part), (size_t)m * 32 * 4);
  if (e == hipSuccess) e = launch_fold_ln(dtype16, d_w32, d_gamma, d_beta, d_bias, wf, cs, bf, n, C, s);
  if (e == hipSuccess) e = launch_rowsums(d_x, dtype16, C, part, m, C, s);
  if (e == hipSuccess) e = launch_permute_qkv_obj(wf, bf, cs, wp, bfp, csp, C, s);
  for (int i = 0; i < (repeats < 1 ? 1 : repeats) && e == hipSuccess; ++i)
    e = launch_qkv_attn_obj(dtype16, d_x, wp, bfp, csp, part, 1, d_mask, mask_dtype, d_out, n_img, l, heads, &t_debug_opts, s,
                            reinterpret_cast<unsigned long long*>(d_trace));
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  (void)hipFree(wf); (void)hipFree(wp); (void)hipFree(cs); (void)hipFree(bf); (void)hipFree(csp); (void)hipFree(bfp);
  (void)hipFree(part);
  return dbg(e);
}

int oake_debug_layernorm(const void* d_x, int x_dtype, const float* d_gamma, const float* d_beta,
                         void* d_y, int rows, int c, int dtype16, void* stream) {
  return dbg(launch_layernorm(dtype16, d_x, x_dtype, c, d_gamma, d_beta, d_y, rows, c,
                              reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_attention(const void* d_qkv, void* d_out, int n, int l, int heads, int dtype16,
                         void* stream) {
  return dbg(launch_attention(dtype16, d_qkv, d_out, n, l, heads, 0, reinterpret_cast<hipStream_t>(stream),
                              nullptr, nullptr, 0, nullptr, &t_debug_opts));
}

int oake_debug_attention_objects(const void* d_qkv, const void* d_qkv_y, const void* d_mask, int mask_dtype,
                                 void* d_out, void* d_out_y, int n, int l, int heads, int dtype16, void* stream) {
  if (!d_qkv || !d_qkv_y || !d_mask || !d_out || !d_out_y) return OAKE_ERR_INVALID;
  if (!attention_fuses_object_token(l, &t_debug_opts)) return OAKE_ERR_UNSUPPORTED;
  return dbg(launch_attention(dtype16, d_qkv, d_out, n, l, heads, 0, reinterpret_cast<hipStream_t>(stream), d_qkv_y,
                              d_mask, mask_dtype, d_out_y, &t_debug_opts));
}

int oake_debug_attn_out(const void* d_qkv, const void* d_w, const float* d_bias, void* d_x, float* d_rowpart,
                        int n, int l, int heads, int dtype16, void* stream) {
  return oake_debug_attn_out_trace(d_qkv, d_w, d_bias, d_x, d_rowpart, n, l, heads, dtype16, nullptr, 1, stream);
}

int oake_debug_attn_out_trace(const void* d_qkv, const void* d_w, const float* d_bias, void* d_x, float* d_rowpart,
                              int n, int l, int heads, int dtype16, void* d_trace, int repeats, void* stream) {
#if !OAKE_LAB
  // (the kernel lost its A/B — docs/history/round4.md item 4 — and lives in liboake_hip_lab.so only)
  (void)d_qkv; (void)d_w; (void)d_bias; (void)d_x; (void)d_rowpart; (void)n; (void)l; (void)heads; (void)dtype16;
  (void)d_trace; (void)repeats; (void)stream;
  return OAKE_ERR_UNSUPPORTED;
#else
  const int C = heads * 64;
  if (!d_qkv || !d_w || !d_bias || !d_x || !d_rowpart || n < 0) return OAKE_ERR_INVALID;
  if (!attn_out_supported(l, heads, C)) return OAKE_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void* wp = nullptr;
  if (hipMalloc(&wp, (size_t)C * C * 2) != hipSuccess) return OAKE_ERR_HIP;
  hipError_t e = launch_permute_out_w(dtype16, d_w, wp, s);
  for (int i = 0; i < repeats && e == hipSuccess; ++i)
    e = launch_attn_out(dtype16, d_qkv, wp, d_bias, d_x, d_rowpart, n, l, s,
                        reinterpret_cast<unsigned long long*>(d_trace));
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  (void)hipFree(wp);
  return dbg(e);
#endif
}

int oake_debug_tr_read(const uint16_t* d_in, uint16_t* d_out, void* stream) {
  return dbg(launch_tr_read_probe(d_in, d_out, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_cu_census(uint32_t* d_out, int nblocks, int hold_us, void* stream) {
  if (!d_out || nblocks < 1 || hold_us < 0) return OAKE_ERR_INVALID;
  return dbg(launch_cu_census(d_out, nblocks, hold_us, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_mfma_probe(const void* d_frags16, float* d_sink, int iters, double* flop, void* stream) {
  if (d_frags16 == nullptr || d_sink == nullptr || iters < 1) return OAKE_ERR_INVALID;
  return dbg(launch_mfma_probe(d_frags16, d_sink, iters, flop, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_mfma_probe_order(const void* d_frags16, float* d_sink, int iters, int order, double* flop, void* stream) {
  if (d_frags16 == nullptr || d_sink == nullptr || iters < 1 || order < 0 || order > 3) return OAKE_ERR_INVALID;
  return dbg(launch_mfma_probe_order(d_frags16, d_sink, iters, order, flop, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_mfma_probe_32x32(const void* d_frags16, float* d_sink, int iters, double* flop, void* stream) {
  if (d_frags16 == nullptr || d_sink == nullptr || iters < 1) return OAKE_ERR_INVALID;
  return dbg(launch_mfma_probe32(d_frags16, d_sink, iters, flop, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_set_gemm_variant(int variant) {
  if (variant < -2 || !gemm_variant_supported(variant)) return OAKE_ERR_UNSUPPORTED;
  t_debug_opts.gemm_variant = variant;
  return OAKE_OK;
}

int oake_debug_gemm_resid16(const void* d_a, const void* d_w, const float* d_bias, void* d_x,
                            float* d_rowpart, int m, int n, int k, int dtype16, void* stream) {
  GemmArgs a{};
  a.A = d_a; a.W = d_w; a.bias = d_bias; a.out = d_x; a.M = m; a.N = n; a.K = k; a.ldo = n;
  a.opts = &t_debug_opts;
  a.rowpart_out = gemm_uses_persistent(m, n, k, &t_debug_opts) ? d_rowpart : nullptr;
  return dbg(launch_gemm(dtype16, EPI_RESID16, a, reinterpret_cast<hipStream_t>(stream)));
}

int oake_debug_set_gemm_panel(int panel) {
  t_debug_opts.gemm_panel = panel;
  return OAKE_OK;
}

int oake_debug_set_qkv_walk(int heads_per_block) {
  if (heads_per_block < 0 || heads_per_block > 32) return OAKE_ERR_INVALID;
  t_debug_opts.qkv_walk = heads_per_block;
  return OAKE_OK;
}

int oake_debug_set_gemm_trace(void* d_trace) {
  t_debug_opts.gemm_trace = reinterpret_cast<unsigned long long*>(d_trace);
  return OAKE_OK;
}

int oake_debug_set_attention_variant(int variant) {
  if (variant < 0 || variant > 255 || !attention_variant_supported(variant)) return OAKE_ERR_UNSUPPORTED;
  t_debug_opts.attention_variant = variant;
  return OAKE_OK;
}

int oake_debug_lab_build(void) { return OAKE_LAB; }

int oake_set_option(oake_handle* h, int option, int value) {
  if (!h) return OAKE_ERR_INVALID;
  switch (option) {
    case OAKE_OPT_CLS_LAST: h->cls_last = value ? 1 : 0; return OAKE_OK;
    case OAKE_OPT_GEMM_VARIANT:
      if (value < -2 || !gemm_variant_supported(value))
        return fail(h, OAKE_ERR_INVALID, "gemm variant " + std::to_string(value) + " is not in this build (production: -1, 0, 4, 5, 13; "
                    "the experiments live in liboake_hip_lab.so)");
      h->opts.gemm_variant = value;
      return OAKE_OK;
    case OAKE_OPT_GEMM_PANEL:
      if (value < -64 || value > 64) return fail(h, OAKE_ERR_INVALID, "gemm_panel must be in -64 .. 64");
      h->opts.gemm_panel = value;
      return OAKE_OK;
    case OAKE_OPT_ATTENTION_VARIANT:
      if (value < 0 || value > 255 || !attention_variant_supported(value))
        return fail(h, OAKE_ERR_INVALID, "attention variant " + std::to_string(value) + " is not in this build (production: 31)");
      h->opts.attention_variant = value;
      return OAKE_OK;
    case OAKE_OPT_PATCH_DIRECT:
      if (value < 0 || value > (OAKE_LAB ? 2 : 1))
        return fail(h, OAKE_ERR_INVALID, "patch_direct must be 0 or 1 (2: lab build only)");
      h->patch_direct = value;
      return OAKE_OK;
    case OAKE_OPT_CU_COUNT:
      if (value < 0 || value > 4096) return fail(h, OAKE_ERR_INVALID, "cu_count must be in 0 .. 4096");
      h->opts.cu_count = value;
      return OAKE_OK;
    case OAKE_OPT_FUSE_ATTN_OUT:
#if OAKE_LAB
      // the permuted copies of W_out (C x C 16-bit per layer) exist only once the option has been switched on,
      // and only where the kernel can run (the REAL sequence length: never at L = 197)
      if (value && !h->text && h->xdt != DT_F32 && attn_out_supported(h->tokens, h->cfg.heads, h->cfg.width)) {
        HIP_TRY(h, hipSetDevice(h->device));
        const size_t C = h->cfg.width;
        for (auto& l : h->layers)
          if (!l.out_wp) {
            HIP_TRY(h, hipMalloc(&l.out_wp, C * C * 2));
            HIP_TRY(h, launch_permute_out_w(h->dt16, l.out_w, l.out_wp, 0));
          }
        HIP_TRY(h, hipStreamSynchronize(0));
      }
      h->fuse_attn_out = value ? 1 : 0;
      return OAKE_OK;
#else
      if (value) return fail(h, OAKE_ERR_INVALID, "fuse_attn_out: the fused attention + out_proj kernel is in "
                             "liboake_hip_lab.so only (measured slower: docs/history/round4.md item 4)");
      return OAKE_OK;
#endif
    case OAKE_OPT_FUSE_QKV_ATTN: {
      if (value < 0 || value > 2) return fail(h, OAKE_ERR_INVALID, "OAKE_OPT_FUSE_QKV_ATTN: 0, 1 or 2");
#if !OAKE_LAB
      if (value == 2)
        return fail(h, OAKE_ERR_INVALID, "OAKE_OPT_FUSE_QKV_ATTN = 2 (the three-image form, csrc/qkv_attn.hip) is in the lab "
                                         "build liboake_hip_lab.so only");
#endif
      const bool was_obj = qkv_perm_is_obj(h);
      h->fuse_qkv_attn = value;
      if (qkv_perm_is_obj(h) != was_obj) h->qkv_perm = false;  // (the other form's column order: permuted again on the next pass)
      return OAKE_OK;
    }
    case OAKE_OPT_QKV_WALK:
      if (value < 0 || value > 32) return fail(h, OAKE_ERR_INVALID, "OAKE_OPT_QKV_WALK: 0 (group-major) or heads per head block, 1 .. 32");
      h->opts.qkv_walk = value;
      return OAKE_OK;
    case OAKE_OPT_PASS_CROPS:
      if (h->text) return fail(h, OAKE_ERR_INVALID, "pass_crops: vision handles only");
      if (value < 1) return fail(h, OAKE_ERR_INVALID, "pass_crops must be >= 1");
      h->cfg.max_batch = std::min(value, h->pass_cap);  // (a bound: never above what the workspace was created for)
      return OAKE_OK;
    default: return fail(h, OAKE_ERR_INVALID, "unknown option " + std::to_string(option));
  }
}

int oake_get_option(const oake_handle* h, int option, int* value) {
  if (!h || !value) return OAKE_ERR_INVALID;
  switch (option) {
    case OAKE_OPT_CLS_LAST: *value = h->cls_last; return OAKE_OK;
    case OAKE_OPT_GEMM_VARIANT: *value = h->opts.gemm_variant; return OAKE_OK;
    case OAKE_OPT_GEMM_PANEL: *value = h->opts.gemm_panel; return OAKE_OK;
    case OAKE_OPT_ATTENTION_VARIANT: *value = h->opts.attention_variant; return OAKE_OK;
    case OAKE_OPT_PATCH_DIRECT: *value = h->patch_direct; return OAKE_OK;
    case OAKE_OPT_CU_COUNT: *value = h->opts.cu_count; return OAKE_OK;
    case OAKE_OPT_FUSE_ATTN_OUT: *value = h->fuse_attn_out; return OAKE_OK;
    case OAKE_OPT_PASS_CROPS: *value = h->cfg.max_batch; return OAKE_OK;
    case OAKE_OPT_FUSE_QKV_ATTN: *value = h->fuse_qkv_attn; return OAKE_OK;
    case OAKE_OPT_QKV_WALK: *value = h->opts.qkv_walk; return OAKE_OK;
    default: return OAKE_ERR_INVALID;
  }
}

// Test hook: a 16-bit matmul weight as it sits on the device (after the f32 -> 16-bit upload, the 1/8 scale
// of the q rows, the transposition of the projection; "<key>#folded": the gamma-folded copy).
int oake_debug_read_weight16(oake_handle* h, const char* name, uint16_t* h_out, size_t numel) {
  if (!h || !name || !h_out) return OAKE_ERR_INVALID;
  HIP_TRY(h, hipSetDevice(h->device));
  int rc = check_ready(h);
  if (rc) return rc;
  std::string key(name);
  bool folded = false;
  const size_t hash = key.find('#');
  if (hash != std::string::npos) {
    folded = key.substr(hash) == "#folded";
    key = key.substr(0, hash);
  }
  const size_t C = h->cfg.width, F = h->cfg.mlp_dim, E = h->cfg.embed_dim;
  const void* src = nullptr;
  size_t n = 0;
  if (!h->text && key == "visual.conv1.weight") { src = h->conv_w; n = C * h->kpatch; }
  else if (key == (h->text ? "text_projection" : "visual.proj")) { src = h->proj; n = C * E; }
  else {
    const std::string prefix = h->text ? "transformer.resblocks." : "visual.transformer.resblocks.";
    if (key.compare(0, prefix.size(), prefix) != 0) return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "unknown tensor: " + key);
    const size_t dot = key.find('.', prefix.size());
    if (dot == std::string::npos) return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "unknown tensor: " + key);
    const int l = std::atoi(key.substr(prefix.size(), dot - prefix.size()).c_str());
    if (l < 0 || l >= (int)h->layers.size()) return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "unknown tensor: " + key);
    const std::string leaf = key.substr(dot + 1);
    const LayerW& w = h->layers[l];
    if (leaf == "attn.in_proj_weight") { src = folded ? w.in_wf : w.in_w; n = 3 * C * C; }
    else if (leaf == "attn.out_proj.weight" && !folded) { src = w.out_w; n = C * C; }
    else if (leaf == "mlp.c_fc.weight") { src = folded ? w.fc_wf : w.fc_w; n = F * C; }
    else if (leaf == "mlp.c_proj.weight" && !folded) { src = w.proj_w; n = C * F; }
  }
  if (!src) return fail(h, OAKE_ERR_UNKNOWN_TENSOR, "no 16-bit weight named " + std::string(name));
  if (n != numel) return fail(h, OAKE_ERR_INVALID, key + ": expected " + std::to_string(n) + " elements");
  HIP_TRY(h, hipMemcpy(h_out, src, n * 2, hipMemcpyDeviceToHost));
  return OAKE_OK;
}

}  // extern "C"
