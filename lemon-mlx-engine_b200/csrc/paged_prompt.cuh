// paged_prompt.cuh -- attention of new tokens over the paged cache for many
// query rows per KV head (prompts, chunks, mixed batches) on tcgen05.
//
// The G query heads of a KV head times TT = 128 / G tokens are one 128-row
// tile (row t*G + g), so grouped heads share every K and V tile; an item is
// (sequence, KV head, pair of row tiles), and its keys go in tiles of 128:
//   S = Q K^T         (128 x 128 x D, both operands in shared memory)
//   p = 2^(s - m), l += sum p        (one thread per row)
//   O += P V          (128 x D x 128, P in tensor memory)
// For D = 128 a key tile of one row tile costs 1024 tensor cycles and 128 * 128
// exponentials, 1024 cycles of the SM's special-function unit: the two row
// tiles of a pair take turns, one in the tensor pipe while the other is in
// its softmax, so both units stay busy.
//
// Warps: 0-3 and 4-7 softmax and epilogue of the pair's first and second tile
// (a thread owns a row); 8 issues the MMAs; 9 loads (TMA: one box per page and
// 64 head dims, so the tile in shared memory is the same whatever the page
// size); 10 follows the loads and clears the V rows of a tile that lie past the
// sequence's end (p = 0 there, but 0 * NaN is not 0).
// Tensor memory: S of the two tiles [0, 256), O at 256; P (16-bit) overlays
// the first half of its S, which the softmax has then read.  MMAs issued by
// one thread run in order, so "S(j+1) done" also says that P(j) has been used
// and O is up to date.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 (the old
// maximum stays the reference until then: p <= 256, harmless in fp32 and
// bf16, whose exponents have room), so most tiles touch O in the MMA alone.
//
// Work split: as in the few-row kernel, the 128-key blocks of all items are
// laid end to end and divided evenly over one CTA per SM; items that cross a
// boundary leave fp32 partials that paged_prompt_join_kernel adds in order.
// The division is computed once, by paged_prompt_plan_kernel.
#pragma once
#include "paged.cuh"
#include "sm100.cuh"

namespace lmx {

static constexpr int kPromptThreads = 384;
static constexpr int kPromptRows = 256;  // rows of a pair

struct PromptArgs {
  PagedAttnArgs a;   // nctas = CTAs of the grid; prefix[0] = total blocks; ml / part per slot of 256 rows
  int TT;            // tokens of one row tile
  int4* start;       // [nctas] sequence, head, pair, block where a CTA begins
};
struct PromptMaps {
  CUtensorMap q, k, v;
};

// one pair of row tiles
struct PromptItem {
  int first, nnew, kvlen, len;  // the sequence: packed token, new tokens, rows (and as far as the table reaches)
  int pairs, t0, tn;            // pairs of the sequence; this pair's first token and token count
  int kb, nblk;                 // first 128-key block, blocks
  int lo, hi;                   // keys that any row sees
};
LMX_DEV void prompt_seq(const PromptArgs& p, int s, PromptItem& z) {
  const PagedBatch& b = p.a.b;
  const int q0 = min(max(__ldg(b.q_start + s), 0), b.tokens);
  z.first = q0;
  z.nnew = max(min(__ldg(b.q_start + s + 1), b.tokens) - q0, 0);
  z.kvlen = __ldg(b.kv_len + s);
  z.len = (int)min((int64_t)max(z.kvlen, 0), (int64_t)b.table_stride << p.a.kv.logP);
  z.pairs = (z.nnew + 2 * p.TT - 1) / (2 * p.TT);
}
LMX_DEV void prompt_pair(const PromptArgs& p, int pair, PromptItem& z) {
  z.t0 = pair * 2 * p.TT;
  z.tn = min(2 * p.TT, z.nnew - z.t0);
  const int p0 = z.kvlen - z.nnew + z.t0;  // position of the pair's first token
  z.hi = max(0, min(z.len, p0 + z.tn));
  z.lo = p.a.window > 0 ? min(max(0, p0 - p.a.window + 1), z.hi) : 0;
  z.kb = z.lo >> 7;
  z.nblk = max(1, ((z.hi + 127) >> 7) - z.kb);
}

// Blocks before each sequence, and where each CTA begins.
__global__ void __launch_bounds__(1024) paged_prompt_plan_kernel(PromptArgs p) {
  __shared__ int64_t pre[kPagedMaxSeqs + 1];
  __shared__ int64_t wsum[32];
  grid_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seqs = p.a.b.seqs;
  for (int s = warp; s < seqs; s += 32) {
    PromptItem z;
    prompt_seq(p, s, z);
    if (lane == 0 && z.nnew > 0 && z.kvlen > z.len) atomicExch(p.a.err, kPagedErr);
    int64_t n = 0;
    for (int i = lane; i < z.pairs; i += 32) {
      prompt_pair(p, i, z);
      n += z.nblk;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
    if (lane == 0) pre[s + 1] = n * p.a.kv.Hk;
  }
  if (tid == 0) pre[0] = 0;
  __syncthreads();
  // inclusive scan, two entries per thread
  const int i0 = 2 * tid + 1, i1 = i0 + 1;
  const int64_t v0 = i0 <= seqs ? pre[i0] : 0, v1 = i1 <= seqs ? pre[i1] : 0;
  int64_t v = v0 + v1;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  if (lane == 31) wsum[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += wsum[w];
  if (i0 <= seqs) pre[i0] = v - v1;
  if (i1 <= seqs) pre[i1] = v;
  __syncthreads();
  const int64_t total = pre[seqs];
  if (tid == 0) p.a.prefix[0] = total;
  const int n = (int)(total < p.a.nctas ? total : p.a.nctas);
  for (int c = warp; c < n; c += 32) {
    const int64_t at = total * c / n;
    int s = 0, e = seqs;
    while (e - s > 1) {
      const int mid = (s + e) / 2;
      if (pre[mid] <= at) s = mid;
      else e = mid;
    }
    while (pre[s + 1] <= at) ++s;
    PromptItem z;
    prompt_seq(p, s, z);
    const int64_t per = (pre[s + 1] - pre[s]) / p.a.kv.Hk, loc = at - pre[s];
    const int h = (int)(loc / per);
    int rem = (int)(loc % per);
    for (int base = 0;; base += 32) {  // the pair that holds block rem of this head
      int nb = 0;
      if (base + lane < z.pairs) {
        prompt_pair(p, base + lane, z);
        nb = z.nblk;
      }
      int inc = nb;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, inc > rem);
      if (past) {
        const int l = __ffs(past) - 1;
        const int before = __shfl_sync(0xffffffffu, inc - nb, l);
        if (lane == 0) p.start[c] = make_int4(s, h, base + l, rem - before);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

// A CTA's walk over its blocks: one segment (item, blocks [b0, b1)) at a time.
struct PromptWalk {
  int seq, h, pair, b0, b1;
  int64_t left;  // blocks from b0 to the CTA's end
  PromptItem z;
  bool first;

  LMX_DEV void begin(const PromptArgs& p) {
    const int64_t total = p.a.prefix[0], n = total < p.a.nctas ? total : p.a.nctas;
    left = 0;
    if (blockIdx.x >= n) return;
    left = total * (blockIdx.x + 1) / n - total * blockIdx.x / n;
    const int4 s = p.start[blockIdx.x];
    seq = s.x; h = s.y; pair = s.z; b0 = s.w;
    prompt_seq(p, seq, z);
    prompt_pair(p, pair, z);
    b1 = (int)min((int64_t)z.nblk, b0 + left);
    first = true;
  }
  LMX_DEV bool live() const { return left > 0; }
  LMX_DEV void next(const PromptArgs& p) {
    left -= b1 - b0;
    first = false;
    if (left <= 0) return;
    b0 = 0;
    if (++pair == z.pairs) {
      pair = 0;
      if (++h == p.a.kv.Hk) {
        h = 0;
        do prompt_seq(p, ++seq, z);
        while (z.nnew == 0);
      }
    }
    prompt_pair(p, pair, z);
    b1 = (int)min((int64_t)z.nblk, left);
  }
  LMX_DEV bool second(const PromptArgs& p) const { return z.tn > p.TT; }  // the pair's second tile has rows
  LMX_DEV bool whole() const { return b0 == 0 && b1 == z.nblk; }
};

// Bounded wait, in line (a call would spill the softmax's registers): the
// hardware suspends the thread for up to a millisecond per try; gives up after
// 4 s or 2^20 tries and sets the error word.
LMX_DEV bool prompt_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
#pragma unroll 1
  for (int i = 0; i < (1 << 20); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (global_ns() - t0 > 4000000000ull) break;
  }
  atomicExch(err, code);
  return false;
}
LMX_DEV bool prompt_warp_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  return __all_sync(0xffffffffu, prompt_wait(bar, parity, err, code));
}

LMX_DEV void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
LMX_DEV void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// D[tmem] (+)= A[smem] * B[smem]^T
LMX_DEV void umma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
LMX_DEV void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
LMX_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
LMX_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
LMX_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
LMX_DEV void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
LMX_DEV void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// V is the B operand with its N index (head dims) contiguous: 64-value blocks
// of 128 bytes (leading byte offset: from one block of 64 head dims to the
// next, 128 keys * 128 bytes), 8-key groups 1024 bytes apart.
LMX_DEV uint64_t umma_desc_v(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <int D>
struct PromptSmem {
  static constexpr int TILE = 128 * D * 2;            // one tile of Q, K or V
  static constexpr int NS = D == 128 ? 5 : 8;         // K / V stages
  static constexpr int BYTES = 2 * TILE + NS * TILE + 1024 + 256;
};

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    paged_prompt_kernel(const __grid_constant__ PromptMaps mp, const __grid_constant__ PromptArgs p) {
  using SM = PromptSmem<D>;
  constexpr int TILE = SM::TILE, NS = SM::NS, NH = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* Qs = smem;
  uint8_t* KV = smem + 2 * TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(KV + NS * TILE);
  uint64_t *q_full = bars, *q_free = bars + 1, *vfix = bars + 2, *s_full = bars + 3, *p_ready = bars + 5,
           *o_full = bars + 7, *o_free = bars + 9, *drain = bars + 11, *kv_full = bars + 12, *kv_free = kv_full + NS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_free + NS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(vfix, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 4);
      mbar_init(o_full + i, 1);
      mbar_init(o_free + i, 4);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_free + i, 2);  // the MMAs' commit and warp 10
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_wait();
  grid_launch_dependents();
  unsigned* err = p.a.err;
  PromptWalk w;

  if (warp < 8) {
    // ------------------------- softmax and epilogue -------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int tile = warp >> 2;  // of the pair
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
    const uint32_t tS = tmem + lanes + tile * 128, tO = tmem + lanes + 256 + tile * D;
    const int r = (warp & 3) * 32 + lane;               // row of the tile
    const int G = p.a.G;
    const float scale2 = p.a.scale2;
    uint32_t ps = 0, po = 0;  // parities of s_full, o_full
    bool ok = true;
    for (w.begin(p); ok && w.live(); w.next(p)) {
      if (tile == 1 && !w.second(p)) continue;
      const int t = r / G, tok = w.z.t0 + tile * p.TT + t;  // token of the sequence
      const bool row = t < p.TT && tok < w.z.nnew;
      const int pos = w.z.kvlen - w.z.nnew + tok;
      // rows of nobody are not stored; they count as seeing everything, so that
      // they do not send their warp through the masks
      const int khi = row ? min(pos + 1, w.z.len) : 1 << 30;
      const int klo = row && p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0;
      float m = -INFINITY, l = 0.0f;
      for (int b = w.b0; b < w.b1; ++b) {
        ok = prompt_warp_wait(s_full + tile, ps, err, 0x45u);
        if (!ok) break;
        ps ^= 1;
        tmem_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(tS + 32 * i, s + 32 * i);
        tmem_wait_ld();
        const int key = (w.z.kb + b) << 7;
        if (!__all_sync(0xffffffffu, key + 128 <= khi && key >= klo)) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key + i >= khi || key + i < klo) s[i] = 0xff800000u;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 128; ++i) mx = fmaxf(mx, __uint_as_float(s[i]));
        mx *= scale2;
        if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
          const float mn = fmaxf(m, mx);
          if (b > w.b0) {
            const float al = mn == -INFINITY ? 1.0f : ex2f(m - mn);
            l *= al;
#pragma unroll
            for (int i = 0; i < D; i += 16) {
              float o[16];
              uint32_t u[16];
              tmem_ld16(tO + i, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(o[k] * al);
              tmem_st16(tO + i, u);
            }
          }
          m = mn;
        }
        const float ms = m == -INFINITY ? 0.0f : -m;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p0 = ex2f(__fmaf_rn(__uint_as_float(s[32 * h + 2 * i]), scale2, ms));
            const float p1 = ex2f(__fmaf_rn(__uint_as_float(s[32 * h + 2 * i + 1]), scale2, ms));
            sum[i & 1] += p0;
            sum[2 + (i & 1)] += p1;
            pk[i] = pk_bf2(p0, p1);
          }
          tmem_st16(tS + 16 * h, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + tile);
      }
      if (!ok) break;
      ok = prompt_warp_wait(o_full + tile, po, err, 0x46u);
      if (!ok) break;
      po ^= 1;
      tmem_fence_after();
      const int head = w.h * G + r % G;
      if (w.whole()) {
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        bf16_t* op = p.a.out + (int64_t)(w.z.first + tok) * p.a.ldo + (int64_t)head * D;
#pragma unroll
        for (int i = 0; i < D; i += 32) {
          uint32_t o[32];
          tmem_ld32(tO + i, o);
          tmem_wait_ld();
          if (row)
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[k + e]) * inv;
              *reinterpret_cast<uint4*>(op + i + k) = bf8_pack(y);
            }
        }
        if (row && p.a.lse)
          p.a.lse[(int64_t)(w.z.first + tok) * p.a.heads + head] =
              l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
      } else {
        const int64_t slot = 2 * (int64_t)blockIdx.x + (w.first ? 0 : 1);
        float4* pp = reinterpret_cast<float4*>(p.a.part) + slot * (D / 4) * kPromptRows + tile * 128 + r;
#pragma unroll
        for (int i = 0; i < D; i += 32) {
          uint32_t o[32];
          tmem_ld32(tO + i, o);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            pp[(i + k) / 4 * kPromptRows] = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]),
                                                        __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
        }
        *reinterpret_cast<float2*>(p.a.ml + (slot * kPromptRows + tile * 128 + r) * 2) = make_float2(m, l);
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free + tile);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8 && lane == 0) {
      // ------------------------------ MMA issue ------------------------------
      // A and B bf16 (formats 1), D fp32; M = 128
      const uint32_t iS = umma_idesc_bf16(128), iO = umma_idesc_bf16(D) | (1u << 16);  // B of P V is N-major
      uint32_t pq = 0, pfix = 0, pp[2] = {0, 0}, pof[2] = {1, 1};
      int st = 0;
      uint32_t pst = 0;  // ring stage and parity of kv_full
      const uint32_t qa = smem_u32(Qs), ka = smem_u32(KV);
      auto mma_s = [&](int tile, int stage) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(tmem + tile * 128, umma_desc_sw128(qa + tile * TILE + (k >> 2) * 16384 + (k & 3) * 32),
                  umma_desc_sw128(ka + stage * TILE + (k >> 2) * 16384 + (k & 3) * 32), iS, k > 0);
      };
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, unsigned code) {
        ok = ok && prompt_wait(bar, parity, err, code);
        return ok;
      };
      auto step = [&](int& s, uint32_t& par) {
        if (++s == NS) { s = 0; par ^= 1; }
      };
      for (w.begin(p); ok && w.live(); w.next(p)) {
        const int tiles = w.second(p) ? 2 : 1, n = w.b1 - w.b0;
        if (!wait(q_full, pq, 0x47u) || !wait(kv_full + st, pst, 0x48u)) break;
        pq ^= 1;
        tmem_fence_after();
        for (int i = 0; i < tiles; ++i) {
          mma_s(i, st);
          umma_commit(s_full + i);
        }
        umma_commit(kv_free + st);
        step(st, pst);
        if (n == 1) umma_commit(q_free);
        for (int j = 0; j < n && ok; ++j) {
          // stages: V(j) at st, K(j+1) after it
          const int sv = st;
          int sk = st;
          uint32_t pk = pst;
          step(sk, pk);
          if (!wait(kv_full + sv, pst, 0x48u)) break;
          const bool tail = ((w.z.kb + w.b0 + j + 1) << 7) > w.z.len;
          if (tail) {
            if (!wait(vfix, pfix, 0x49u)) break;
            pfix ^= 1;
          }
          if (j + 1 < n && !wait(kv_full + sk, pk, 0x48u)) break;
          for (int i = 0; i < tiles; ++i) {
            if (!wait(p_ready + i, pp[i], 0x4Au)) break;
            pp[i] ^= 1;
            if (j == 0) {  // O of the previous item has been read
              if (!wait(o_free + i, pof[i], 0x4Bu)) break;
              pof[i] ^= 1;
            }
            tmem_fence_after();
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_ts_bf16(tmem + 256 + i * D, tmem + i * 128 + k * 8, umma_desc_v(ka + sv * TILE + k * 2048), iO,
                           j > 0 || k > 0);
            if (j + 1 < n) {
              mma_s(i, sk);
              umma_commit(s_full + i);
            } else {
              umma_commit(o_full + i);
            }
          }
          if (!ok) break;
          umma_commit(kv_free + sv);
          step(st, pst);
          if (j + 1 < n) {
            umma_commit(kv_free + sk);
            step(st, pst);
          }
          if (j + 2 == n) umma_commit(q_free);  // the last S is issued
        }
      }
      if (!ok) {  // a wait gave up: let the issued MMAs finish before the memory goes
        umma_commit(drain);
        prompt_wait(drain, 0, err, 0x4Eu);
      }
    } else if (warp == 9) {
      // -------------------------------- loads --------------------------------
      const int P = p.a.kv.P, rows = min(P, 128), nbox = 128 / rows;
      const int qbytes = p.TT * p.a.G * 128 * NH;
      int st = 0;
      uint32_t pst = 1, pq = 1;
      int issued = 0;
      bool ok = true, started = false;
      for (w.begin(p); ok && w.live(); w.next(p)) {
        const int tiles = w.second(p) ? 2 : 1;
        ok = prompt_warp_wait(q_free, pq, err, 0x4Cu);
        if (!ok) break;
        pq ^= 1;
        started = true;
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * qbytes));
          for (int i = 0; i < tiles; ++i)
            for (int h = 0; h < NH; ++h)
              tma_load_3d(Qs + i * TILE + h * 16384, &mp.q, h * 64, w.h * p.a.G, w.z.first + w.z.t0 + i * p.TT, q_full);
        }
        for (int b = w.b0; b < w.b1 && ok; ++b) {
          const int key = (w.z.kb + b) * 128 + lane * rows;
          int page = p.a.kv.pages;  // out of range: the box reads as zeros
          if (lane < nbox && key < w.z.hi && key + rows > w.z.lo) {
            page = __ldg(p.a.b.table + (int64_t)w.seq * p.a.b.table_stride + (key >> p.a.kv.logP));
            if ((unsigned)page >= (unsigned)p.a.kv.pages) {
              atomicExch(err, kPagedErr);
              page = p.a.kv.pages;
            }
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = prompt_warp_wait(kv_free + st, pst, err, 0x4Du);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(kv_full + st, (uint32_t)TILE);
            __syncwarp();
            if (lane < nbox)
              for (int h = 0; h < NH; ++h)
                tma_load_4d(KV + st * TILE + h * 16384 + lane * rows * 128, kv ? &mp.v : &mp.k, h * 64, key & (P - 1),
                            w.h, page, kv_full + st);
            ++issued;
            if (++st == NS) { st = 0; pst ^= 1; }
          }
        }
      }
      // leave no copy in flight behind, also where a wait gave up
      for (int k = max(0, issued - NS); k < issued; ++k)
        prompt_wait(kv_full + k % NS, (uint32_t)((k / NS) & 1), err, 0x4Eu);
      if (started) prompt_wait(q_full, pq, err, 0x4Eu);
    } else if (warp == 10) {
      // ------------------ V rows past the sequence's end := 0 ------------------
      int st = 0;
      uint32_t pst = 0;
      bool ok = true;
      for (w.begin(p); ok && w.live(); w.next(p)) {
        for (int b = w.b0; b < w.b1 && ok; ++b) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = prompt_warp_wait(kv_full + st, pst, err, 0x4Fu);
            if (!ok) break;
            const int key = (w.z.kb + b) << 7;
            if (kv == 1 && key + 128 > w.z.len) {
              const int from = max(0, w.z.len - key);
              for (int i = lane; i < (128 - from) * 8 * NH; i += 32) {
                const int half = i / ((128 - from) * 8), at = i % ((128 - from) * 8);
                *reinterpret_cast<uint4*>(KV + st * TILE + half * 16384 + from * 128 + at * 16) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(vfix);
            }
            if (lane == 0) mbar_arrive(kv_free + st);
            if (++st == NS) { st = 0; pst ^= 1; }
          }
        }
      }
    }
    __syncwarp();
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Join of the items that several CTAs share.  Grid (nctas, 8): block (c, i)
// joins 32 rows of the item in which CTA c begins, if CTA c is the first to
// begin inside it (so each shared item is joined once, by its second
// contributor).  Partials are added in CTA order.
template <int D>
__global__ void __launch_bounds__(128) paged_prompt_join_kernel(const __grid_constant__ PromptArgs p) {
  grid_wait();
  grid_launch_dependents();
  const int64_t total = p.a.prefix[0], n = total < p.a.nctas ? total : p.a.nctas;
  const int64_t c = blockIdx.x;
  if (c >= n || c == 0) return;
  const int4 s = p.start[c];
  if (s.w == 0) return;                             // begins with its item
  const int64_t i0 = total * c / n - s.w;           // the item's first block
  if (total * (c - 1) / n > i0) return;             // CTA c - 1 begins inside it too
  PromptItem z;
  prompt_seq(p, s.x, z);
  prompt_pair(p, s.z, z);
  const int64_t c1 = ((i0 + z.nblk) * n - 1) / total;  // CTA of its last block
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), tile = row >> 7, r = row & 127;
  const int t = r / p.a.G, tok = z.t0 + tile * p.TT + t;
  if (t >= p.TT || tok >= z.nnew) return;
  const int64_t slot0 = 2 * (c - 1) + (total * (c - 1) / n < i0 ? 1 : 0);
  auto slot_of = [&](int64_t k) { return k == c - 1 ? slot0 : 2 * k; };
  float M = -INFINITY;
  for (int64_t k = c - 1; k <= c1; ++k) M = fmaxf(M, p.a.ml[(slot_of(k) * kPromptRows + row) * 2]);
  const float ms = M == -INFINITY ? 0.0f : M;
  constexpr int V = D / 16;  // float4 per thread: column groups threadIdx / 32 + 4 i
  float4 acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = make_float4(0, 0, 0, 0);
  float L = 0.0f;
  for (int64_t k = c - 1; k <= c1; ++k) {
    const int64_t sl = slot_of(k);
    const float2 ml = *reinterpret_cast<const float2*>(p.a.ml + (sl * kPromptRows + row) * 2);
    const float wt = ex2f(ml.x - ms);
    L = __fmaf_rn(wt, ml.y, L);
    const float4* pp = reinterpret_cast<const float4*>(p.a.part) + sl * (D / 4) * kPromptRows + row;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float4 x = pp[((threadIdx.x >> 5) + 4 * i) * kPromptRows];
      acc[i].x = __fmaf_rn(wt, x.x, acc[i].x);
      acc[i].y = __fmaf_rn(wt, x.y, acc[i].y);
      acc[i].z = __fmaf_rn(wt, x.z, acc[i].z);
      acc[i].w = __fmaf_rn(wt, x.w, acc[i].w);
    }
  }
  const float inv = L == 0.0f ? 0.0f : __fdiv_rn(1.0f, L);
  const int head = s.y * p.a.G + r % p.a.G;
  bf16_t* op = p.a.out + (int64_t)(z.first + tok) * p.a.ldo + (int64_t)head * D;
#pragma unroll
  for (int i = 0; i < V; ++i)
    *reinterpret_cast<uint2*>(op + ((threadIdx.x >> 5) + 4 * i) * 4) =
        make_uint2(pk_bf2(acc[i].x * inv, acc[i].y * inv), pk_bf2(acc[i].z * inv, acc[i].w * inv));
  if (p.a.lse && threadIdx.x < 32)
    p.a.lse[(int64_t)(z.first + tok) * p.a.heads + head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
}

}  // namespace lmx
