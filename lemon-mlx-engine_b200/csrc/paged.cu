// paged.cu -- host launchers and C ABI of the rotary and paged-cache
// operators (include/lmx.h, "Paged KV cache").
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "lmx_internal.h"
#include <cudaTypedefs.h>

#include "paged.cuh"
#include "paged_prompt.cuh"

using namespace lmx;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_kv(const lmx_paged_kv* kv, const char* who) {
  if (!kv) return set_error(LMX_ERR_INVALID, "%s: no cache", who);
  if (kv->bits != 16 && kv->bits != 8 && kv->bits != 4)
    return set_error(LMX_ERR_UNSUPPORTED, "%s: bits=%d (16, 8 or 4)", who, kv->bits);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return set_error(LMX_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", who, kv->head_dim);
  if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
    return set_error(LMX_ERR_UNSUPPORTED, "%s: page_size=%d (16, 32, 64, 128 or 256)", who, kv->page_size);
  if (kv->pages <= 0 || kv->kv_heads <= 0)
    return set_error(LMX_ERR_INVALID, "%s: pages=%d kv_heads=%d", who, kv->pages, kv->kv_heads);
  const int64_t rows = (int64_t)kv->kv_heads * kv->page_size;
  if (kv->page_stride && (kv->page_stride < rows || (kv->bits != 16 && kv->page_stride % 16)))
    return set_error(LMX_ERR_INVALID, "%s: page_stride=%lld for %lld rows", who, (long long)kv->page_stride,
                     (long long)rows);
  const void* need[6] = {kv->k, kv->v, nullptr, nullptr, nullptr, nullptr};
  int n = 2;
  if (kv->bits != 16) {
    const void* q[6] = {kv->k_packed, kv->v_packed, kv->k_scales, kv->k_biases, kv->v_scales, kv->v_biases};
    std::memcpy(need, q, sizeof(q));
    n = 6;
  }
  for (int i = 0; i < n; ++i)
    if (!need[i] || !aligned16(need[i]))
      return set_error(LMX_ERR_INVALID, "%s: cache array %d must be a 16-byte aligned device pointer", who, i);
  return LMX_OK;
}

int check_batch(const lmx_paged_batch* b, const char* who) {
  if (!b) return set_error(LMX_ERR_INVALID, "%s: no batch", who);
  if (b->seqs < 0 || b->tokens < 0 || b->max_new < 0 || b->table_stride < 0)
    return set_error(LMX_ERR_INVALID, "%s: negative size in the batch", who);
  if (b->seqs > kPagedMaxSeqs)
    return set_error(LMX_ERR_UNSUPPORTED, "%s: %d sequences (at most %d)", who, b->seqs, kPagedMaxSeqs);
  if (b->seqs > 0 && b->tokens > 0 && (!b->q_start || !b->kv_len || !b->block_table || b->table_stride == 0))
    return set_error(LMX_ERR_INVALID, "%s: q_start, kv_len and block_table are needed", who);
  return LMX_OK;
}

PagedKv dev_kv(const lmx_paged_kv& kv) {
  PagedKv d;
  d.pages = kv.pages;
  d.P = kv.page_size;
  d.logP = 0;
  while ((1 << d.logP) < kv.page_size) ++d.logP;
  d.Hk = kv.kv_heads;
  d.bits = kv.bits;
  d.pstride = kv.page_stride ? kv.page_stride : (int64_t)kv.kv_heads * kv.page_size;
  d.k = (uint8_t*)(kv.bits == 16 ? kv.k : kv.k_packed);
  d.v = (uint8_t*)(kv.bits == 16 ? kv.v : kv.v_packed);
  d.ks = (bf16_t*)kv.k_scales;
  d.kb = (bf16_t*)kv.k_biases;
  d.vs = (bf16_t*)kv.v_scales;
  d.vb = (bf16_t*)kv.v_biases;
  return d;
}

PagedBatch dev_batch(const lmx_paged_batch& b) {
  return PagedBatch{b.seqs, b.tokens, b.q_start, b.kv_len, b.block_table, b.table_stride};
}

int check_rope(const lmx_rope* r, int head_dim, const char* who) {
  if (!r->cos || !r->sin || !aligned16(r->cos) || !aligned16(r->sin))
    return set_error(LMX_ERR_INVALID, "%s: cos and sin must be 16-byte aligned device pointers", who);
  if (r->positions <= 0 || r->rot_dim <= 0 || r->rot_dim % 16 || r->rot_dim > head_dim)
    return set_error(LMX_ERR_INVALID, "%s: rot_dim=%d (a multiple of 16, at most %d), positions=%d", who, r->rot_dim,
                     head_dim, r->positions);
  return LMX_OK;
}

// token rows of `heads` heads, ld values apart
bool bad_rows(const void* p, int64_t ld, int64_t width) { return !p || !aligned16(p) || ld < width || ld % 8; }

// f(head dim, bits) as compile-time constants
template <typename F>
auto on_cache(int D, int bits, F f) {
  auto on_bits = [&](auto d) {
    return bits == 16  ? f(d, std::integral_constant<int, 16>())
           : bits == 8 ? f(d, std::integral_constant<int, 8>())
                       : f(d, std::integral_constant<int, 4>());
  };
  return D == 64 ? on_bits(std::integral_constant<int, 64>()) : on_bits(std::integral_constant<int, 128>());
}


// A token's `steps` split over wpt warps of `run` steps: one warp a step while
// that is at most 64 warps per SM, longer runs beyond (16 to 128 measure alike).
void warp_runs(int tokens, int steps, int most, int& run, int& wpt) {
  const int64_t warps = (int64_t)device_sms() * 64;
  run = (int)std::min<int64_t>(std::min(steps, most), std::max<int64_t>(1, (int64_t)tokens * steps / warps));
  wpt = (steps + run - 1) / run;
  run = (steps + wpt - 1) / wpt;
}

int grid_of(int64_t blocks, unsigned& grid, const char* who) {
  if (blocks > 0x7fffffff) return set_error(LMX_ERR_UNSUPPORTED, "%s: too many rows", who);
  grid = (unsigned)blocks;
  return LMX_OK;
}

}  // namespace

extern "C" int lmx_rope_table(const lmx_rope_scaling* sc, int positions, int rot_dim, float* cos_out, float* sin_out,
                              void* stream) {
  if (!sc || !cos_out || !sin_out) return set_error(LMX_ERR_INVALID, "rope_table: null argument");
  const int half = rot_dim / 2;
  if (rot_dim <= 0 || rot_dim % 16 || half > 128 || positions <= 0 || (int64_t)positions * half > 0x7fffffff)
    return set_error(LMX_ERR_INVALID, "rope_table: rot_dim=%d (a multiple of 16, at most 256), positions=%d", rot_dim,
                     positions);
  if (sc->kind < LMX_ROPE_PLAIN || sc->kind > LMX_ROPE_YARN)
    return set_error(LMX_ERR_UNSUPPORTED, "rope_table: kind=%d", sc->kind);
  if (!(sc->theta > 0) || (sc->kind != LMX_ROPE_PLAIN && !(sc->factor >= 1)))
    return set_error(LMX_ERR_INVALID, "rope_table: theta=%g factor=%g", sc->theta, sc->factor);
  if (sc->kind >= LMX_ROPE_LLAMA3 && !(sc->low > 0 && sc->high > sc->low && sc->orig_positions > 0))
    return set_error(LMX_ERR_INVALID, "rope_table: low=%g high=%g orig_positions=%g", sc->low, sc->high,
                     sc->orig_positions);
  if (sc->kind == LMX_ROPE_YARN && !(sc->theta > 1))
    return set_error(LMX_ERR_INVALID, "rope_table: theta=%g", sc->theta);
  RopeFreqs fr;
  double mul = 1.0;
  const double two_pi = 6.283185307179586476925;
  double r_lo = 0, r_hi = 1;
  if (sc->kind == LMX_ROPE_YARN) {
    // the (fractional) pair that turns n times within the original context
    auto pair_of = [&](double n) {
      return rot_dim * std::log(sc->orig_positions / (n * two_pi)) / (2 * std::log(sc->theta));
    };
    r_lo = std::fmax(std::floor(pair_of(sc->high)), 0.0);
    r_hi = std::fmin(std::ceil(pair_of(sc->low)), (double)rot_dim - 1);
    if (r_hi - r_lo < 1e-3) r_hi = r_lo + 1e-3;
    mul = sc->attn_factor != 0 ? sc->attn_factor : 0.1 * std::log(sc->factor) + 1.0;
  }
  for (int i = 0; i < half; ++i) {
    const double f = std::pow(sc->theta, -2.0 * i / rot_dim);
    double keep = 1.0;  // share of the unstretched frequency
    if (sc->kind == LMX_ROPE_LINEAR) keep = 0.0;
    if (sc->kind == LMX_ROPE_LLAMA3) keep = (sc->orig_positions * f / two_pi - sc->low) / (sc->high - sc->low);
    if (sc->kind == LMX_ROPE_YARN) keep = 1.0 - (i - r_lo) / (r_hi - r_lo);
    keep = std::fmin(std::fmax(keep, 0.0), 1.0);
    fr.f[i] = sc->kind == LMX_ROPE_PLAIN ? f : f * keep + f / sc->factor * (1.0 - keep);
  }
  const int n = positions * half;
  return cuda_check(lmx_launch(rope_table_kernel, dim3((unsigned)(((int64_t)n + 255) / 256)), dim3(256), 0,
                               (cudaStream_t)stream, true, fr, mul, positions, half, cos_out, sin_out),
                    "rope_table: launch");
}

extern "C" int lmx_rope_apply(const lmx_rope* rope, const void* x, int64_t ldx, const int32_t* pos, int tokens,
                              int heads, int head_dim, int inverse, void* y, int64_t ldy, void* stream) {
  if (!rope) return set_error(LMX_ERR_INVALID, "rope: no tables");
  if (tokens < 0 || heads < 0 || head_dim <= 0 || head_dim % 16 || head_dim > 256)
    return set_error(LMX_ERR_INVALID, "rope: tokens=%d heads=%d head_dim=%d (a multiple of 16, at most 256)", tokens,
                     heads, head_dim);
  int rc = check_rope(rope, head_dim, "rope");
  if (rc) return rc;
  if (tokens == 0 || heads == 0) return LMX_OK;
  const int64_t width = (int64_t)heads * head_dim;
  if (!pos || bad_rows(x, ldx, width) || bad_rows(y, ldy, width) || (x == y && ldx != ldy))
    return set_error(LMX_ERR_INVALID,
                     "rope: x and y must be 16-byte aligned, rows a multiple of 8 values and at least heads * head_dim "
                     "apart (in place: equally far)");
  RopeArgs a{rope->cos, rope->sin, rope->positions, rope->rot_dim, rope->interleaved, inverse, (const bf16_t*)x, ldx,
             pos,       tokens,    heads,           head_dim,      (bf16_t*)y,        ldy,     device_error_word()};
  const int hpt = 4;
  const int64_t threads = (int64_t)tokens * ((heads + hpt - 1) / hpt) * (head_dim / 16);
  unsigned grid;
  if ((rc = grid_of((threads + 255) / 256, grid, "rope"))) return rc;
  return cuda_check(lmx_launch(rope_kernel<hpt>, dim3(grid), dim3(256), 0, (cudaStream_t)stream, true, a),
                    "rope: launch");
}

extern "C" int lmx_paged_append(const lmx_paged_kv* kv, const lmx_paged_batch* batch, const lmx_rope* rope,
                                const void* q, const void* k, const void* v, int64_t ld, int heads,
                                const void* q_norm, const void* k_norm, float eps, void* q_out, int64_t ldq_out,
                                void* stream) {
  int rc = check_kv(kv, "paged_append");
  if (!rc) rc = check_batch(batch, "paged_append");
  if (!rc && rope) rc = check_rope(rope, kv->head_dim, "paged_append");
  if (rc) return rc;
  if (batch->tokens == 0 || batch->seqs == 0) return LMX_OK;
  const int D = kv->head_dim;
  if (heads < 0 || (q == nullptr) != (q_out == nullptr) || (q && heads == 0))
    return set_error(LMX_ERR_INVALID, "paged_append: q and q_out go together (heads=%d)", heads);
  if (!q) heads = 0;
  if (bad_rows(k, ld, (int64_t)kv->kv_heads * D) || bad_rows(v, ld, (int64_t)kv->kv_heads * D) ||
      (q && (bad_rows(q, ld, (int64_t)heads * D) || bad_rows(q_out, ldq_out, (int64_t)heads * D) ||
             (q == q_out && ld != ldq_out))))
    return set_error(LMX_ERR_INVALID,
                     "paged_append: q, k, v and q_out must be 16-byte aligned, rows a multiple of 8 values apart and "
                     "wide enough");
  if ((q_norm == nullptr) != (k_norm == nullptr) || !aligned16(q_norm) || !aligned16(k_norm))
    return set_error(LMX_ERR_INVALID, "paged_append: q_norm and k_norm go together, 16-byte aligned");
  AppendArgs a;
  std::memset(&a, 0, sizeof(a));
  a.kv = dev_kv(*kv);
  a.b = dev_batch(*batch);
  if (rope) {
    a.ct = rope->cos;
    a.st = rope->sin;
    a.positions = rope->positions;
    a.rot = rope->rot_dim;
    a.inter = rope->interleaved;
  }
  a.q = (const bf16_t*)q;
  a.k = (const bf16_t*)k;
  a.v = (const bf16_t*)v;
  a.ld = ld;
  a.heads = heads;
  a.qn = (const bf16_t*)q_norm;
  a.kn = (const bf16_t*)k_norm;
  a.eps = eps;
  a.q_out = (bf16_t*)q_out;
  a.ldqo = ldq_out;
  a.err = device_error_word();
  const int steps = (heads + 2 * kv->kv_heads + 512 / D - 1) / (512 / D);
  warp_runs(batch->tokens, steps, kAppendRun, a.run, a.wpt);
  unsigned grid;
  if ((rc = grid_of(((int64_t)batch->tokens * a.wpt + 3) / 4, grid, "paged_append"))) return rc;
  return cuda_check(on_cache(D, kv->bits, [&](auto d, auto bits) {
                      return lmx_launch(paged_append_kernel<decltype(d)::value, decltype(bits)::value>, dim3(grid),
                                        dim3(128), 0, (cudaStream_t)stream, true, a);
                    }),
                    "paged_append: launch");
}

extern "C" int lmx_paged_gather(const lmx_paged_kv* kv, const lmx_paged_batch* batch, void* k_out, void* v_out,
                                void* stream) {
  int rc = check_kv(kv, "paged_gather");
  if (!rc) rc = check_batch(batch, "paged_gather");
  if (rc) return rc;
  if (!aligned16(k_out) || !aligned16(v_out))
    return set_error(LMX_ERR_INVALID, "paged_gather: k_out and v_out must be 16-byte aligned");
  if (batch->tokens == 0 || batch->seqs == 0 || (!k_out && !v_out)) return LMX_OK;
  GatherArgs a{dev_kv(*kv), dev_batch(*batch), (bf16_t*)k_out, (bf16_t*)v_out, 0, 0, device_error_word()};
  warp_runs(batch->tokens, (2 * kv->kv_heads * kv->head_dim / 16 + 31) / 32, 1 << 20, a.run, a.wpt);
  unsigned grid;
  if ((rc = grid_of(((int64_t)batch->tokens * a.wpt + 3) / 4, grid, "paged_gather"))) return rc;
  return cuda_check(on_cache(kv->head_dim, kv->bits, [&](auto d, auto bits) {
                      return lmx_launch(paged_gather_kernel<decltype(d)::value, decltype(bits)::value>, dim3(grid),
                                        dim3(128), 0, (cudaStream_t)stream, true, a);
                    }),
                    "paged_gather: launch");
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
namespace {

// Query rows per KV head (max_new * heads / kv_heads) from which the prompt
// kernel runs; 0: never.
int g_prompt_min_rows = 33;

struct AttnPlan {
  bool prompt = false;
  int rows = 0;  // query rows of an item
  int nctas = 0;
  size_t start = 0, ml = 0, part = 0, bytes = 0;  // offsets into the scratch
};

template <int D, int BITS, int NT>
int few_rows_ctas(int* n) {
  static int per[64] = {};
  int d = 0;
  cudaGetDevice(&d);
  if (!per[d & 63]) {
    const int most = (kPagedMaxSeqs + 1) * 8;
    int rc = cuda_check(cudaFuncSetAttribute(paged_attn_kernel<D, BITS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, most),
                        "paged_attention: set smem");
    int c = 0;
    if (!rc)
      rc = cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&c, paged_attn_kernel<D, BITS, NT>, 128, most),
                      "paged_attention: occupancy");
    if (rc) return rc;
    per[d & 63] = c > 0 ? c : 1;
  }
  *n = per[d & 63] * device_sms();
  return LMX_OK;
}

// f(head dim, bits, 8-row tiles) as compile-time constants
template <typename F>
int few_rows(int D, int bits, int rows, F f) {
  return on_cache(D, bits, [&](auto d, auto b) {
    return rows == 8 ? f(d, b, std::integral_constant<int, 1>()) : f(d, b, std::integral_constant<int, 2>());
  });
}

int check_attn(const lmx_paged_kv* kv, const lmx_paged_batch* batch, int heads, AttnPlan& p) {
  int rc = check_kv(kv, "paged_attention");
  if (!rc) rc = check_batch(batch, "paged_attention");
  if (rc) return rc;
  if (heads <= 0 || heads % kv->kv_heads || heads / kv->kv_heads > 64)
    return set_error(LMX_ERR_UNSUPPORTED, "paged_attention: heads=%d over kv_heads=%d (a multiple, at most 64 times)",
                     heads, kv->kv_heads);
  const int D = kv->head_dim;
  p.prompt = g_prompt_min_rows > 0 &&
             (int64_t)batch->max_new * (heads / kv->kv_heads) >= g_prompt_min_rows;
  if (p.prompt) {
    p.rows = kPromptRows;
    p.nctas = device_sms();
  } else {
    p.rows = (int64_t)batch->max_new * (heads / kv->kv_heads) <= 8 ? 8 : 16;
    rc = few_rows(D, kv->bits, p.rows, [&](auto d, auto bits, auto nt) {
      return few_rows_ctas<decltype(d)::value, decltype(bits)::value, decltype(nt)::value>(&p.nctas);
    });
  }
  if (rc) return rc;
  auto after = [](size_t at, size_t bytes) { return (at + bytes + 255) / 256 * 256; };
  p.start = 256;  // behind the total
  p.ml = after(p.start, (p.prompt ? (size_t)p.nctas : (size_t)batch->tokens * heads) * sizeof(int4));
  p.part = after(p.ml, (size_t)2 * p.nctas * p.rows * 2 * 4);
  p.bytes = p.part + (size_t)2 * p.nctas * p.rows * D * 4;
  return LMX_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)f;
  }();
  return fn;
}

// Map of `rank` dimensions: bf16 with the 128-byte swizzle (boxes of 64 values
// in the first dimension), or 32-bit words as they are; strides in bytes.
int tensor_map(CUtensorMap* m, const void* base, bool words, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
               const cuuint32_t* box) {
  const auto encode = tensor_map_encoder();
  if (!encode) return set_error(LMX_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult r = encode(m, words ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                            const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            words ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(LMX_ERR_INVALID, "paged_attention: tensor map encode failed (%d)", (int)r);
  return LMX_OK;
}

template <int D, int BITS>
int launch_prompt(const PagedAttnArgs& a, const AttnPlan& pl, cudaStream_t st) {
  PromptArgs p;
  p.a = a;
  p.TT = 128 / a.G;
  p.wide = !((uintptr_t)a.out & 31) && a.ldo % 16 == 0;
  p.cost = PromptSmem<D, BITS>::COST;
  p.start = (int4*)((uint8_t*)a.prefix + pl.start);
  PromptMaps mp;
  const cuuint64_t qd[3] = {D, (cuuint64_t)a.heads, (cuuint64_t)a.b.tokens};
  const cuuint64_t qs[2] = {D * 2, (cuuint64_t)a.ldq * 2};
  const cuuint32_t qb[3] = {64, (cuuint32_t)a.G, (cuuint32_t)p.TT};
  int rc = tensor_map(&mp.q, a.q, false, 3, qd, qs, qb);
  constexpr cuuint64_t row = D * BITS / 8;  // bytes
  const cuuint64_t kd[4] = {BITS == 16 ? D : row / 4, (cuuint64_t)a.kv.P, (cuuint64_t)a.kv.Hk, (cuuint64_t)a.kv.pages};
  const cuuint64_t ks[3] = {row, (cuuint64_t)a.kv.P * row, (cuuint64_t)a.kv.pstride * row};
  const cuuint32_t kb[4] = {BITS == 16 ? 64 : (cuuint32_t)row / 4, (cuuint32_t)(a.kv.P < 128 ? a.kv.P : 128), 1, 1};
  if (!rc) rc = tensor_map(&mp.k, a.kv.k, BITS != 16, 4, kd, ks, kb);
  if (!rc) rc = tensor_map(&mp.v, a.kv.v, BITS != 16, 4, kd, ks, kb);
  if (rc) return rc;
  static bool attr_set[64] = {};
  int d = 0;
  cudaGetDevice(&d);
  constexpr int smem = PromptSmem<D, BITS>::BYTES;
  if (!attr_set[d & 63]) {
    rc = cuda_check(cudaFuncSetAttribute(paged_prompt_kernel<D, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                    "paged_attention: set smem");
    if (rc) return rc;
    attr_set[d & 63] = true;
  }
  rc = cuda_check(lmx_launch(paged_prompt_kernel<D, BITS>, dim3(a.nctas), dim3(prompt_threads(BITS)), smem, st, true, mp, p),
                  "paged_attention: prompt launch");
  if (!rc)
    rc = cuda_check(lmx_launch(paged_prompt_join_kernel<D>, dim3(a.nctas, kPromptRows / 32), dim3(128), 0, st, true, p),
                    "paged_attention: join launch");
  return rc;
}

template <int D, int BITS, int NT>
int launch_few(PagedAttnArgs a, cudaStream_t st) {
  a.keys = PagedStep<D, BITS, NT>::KEYS;
  int rc = cuda_check(lmx_launch(paged_attn_kernel<D, BITS, NT>, dim3(a.nctas), dim3(128), (size_t)(a.b.seqs + 1) * 8, st, true, a),
                      "paged_attention: launch");
  if (rc) return rc;
  unsigned grid;
  if ((rc = grid_of((int64_t)a.b.tokens * a.heads, grid, "paged_attention"))) return rc;
  return cuda_check(lmx_launch(paged_combine_kernel<D>, dim3(grid), dim3(128), 0, st, true, a),
                    "paged_attention: join launch");
}

}  // namespace

extern "C" int lmx_set_paged_prompt_min_rows(int rows) {
  if (rows < 0) return set_error(LMX_ERR_INVALID, "paged_prompt_min_rows %d", rows);
  g_prompt_min_rows = rows;
  return LMX_OK;
}
extern "C" int lmx_paged_prompt_min_rows(void) { return g_prompt_min_rows; }

extern "C" size_t lmx_paged_attention_scratch_bytes(const lmx_paged_kv* kv, const lmx_paged_batch* batch, int heads) {
  AttnPlan p;
  return check_attn(kv, batch, heads, p) ? 0 : p.bytes;
}

extern "C" int lmx_paged_attention(const lmx_paged_kv* kv, const lmx_paged_batch* batch, const void* q, int64_t ldq,
                                   int heads, float scale, int window, void* scratch, size_t scratch_bytes, void* out,
                                   int64_t ldo, float* lse, void* stream) {
  AttnPlan p;
  int rc = check_attn(kv, batch, heads, p);
  if (rc) return rc;
  if (batch->tokens == 0 || batch->seqs == 0) return LMX_OK;
  const int D = kv->head_dim;
  if (bad_rows(q, ldq, (int64_t)heads * D) || bad_rows(out, ldo, (int64_t)heads * D))
    return set_error(LMX_ERR_INVALID,
                     "paged_attention: q and out must be 16-byte aligned, rows a multiple of 8 values and at least "
                     "heads * head_dim apart");
  if (window < 0 || !(scale > 0) || std::isinf(scale))
    return set_error(LMX_ERR_INVALID, "paged_attention: window=%d scale=%g (a positive number)", window, scale);
  if (!scratch || !aligned16(scratch) || scratch_bytes < p.bytes)
    return set_error(LMX_ERR_INVALID, "paged_attention: needs %zu bytes of 16-byte aligned scratch (%zu given)", p.bytes,
                     scratch_bytes);
  PagedAttnArgs a;
  a.kv = dev_kv(*kv);
  a.b = dev_batch(*batch);
  a.q = (const bf16_t*)q;
  a.ldq = ldq;
  a.heads = heads;
  a.G = heads / kv->kv_heads;
  a.scale2 = scale * 1.44269504088896340736f;
  a.window = std::min(window, 1 << 30);  // no position reaches it
  a.out = (bf16_t*)out;
  a.ldo = ldo;
  a.lse = lse;
  a.prefix = (int64_t*)scratch;
  a.ml = (float*)((uint8_t*)scratch + p.ml);
  a.part = (float*)((uint8_t*)scratch + p.part);
  a.rows = p.rows;
  a.shared_by = (int4*)((uint8_t*)scratch + p.start);
  a.nctas = p.nctas;
  a.sms = device_sms();
  a.err = device_error_word();
  cudaStream_t st = (cudaStream_t)stream;
  if (p.prompt)
    return on_cache(D, kv->bits, [&](auto d, auto bits) {
      return launch_prompt<decltype(d)::value, decltype(bits)::value>(a, p, st);
    });
  return few_rows(D, kv->bits, p.rows, [&](auto d, auto bits, auto nt) {
    return launch_few<decltype(d)::value, decltype(bits)::value, decltype(nt)::value>(a, st);
  });
}
