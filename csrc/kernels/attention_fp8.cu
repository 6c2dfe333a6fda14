// Paged GQA attention over the e4m3 KV cache (format: sil/kv_fp8.cuh) for few query rows: one decoded
// token of a sequence, or a short run of tokens.
//
// A unit of work is (sequence, row tile, KV head) with the pages it sees.  A tile is 8 or 16 query
// rows, a row being a (token, query head) pair of the heads that share the KV head.  The products run
// transposed on mma.sync m16n8k16, S^T = K Q^T and O^T = V^T P^T, so that the rows are its n = 8 side:
// up to eight heads to a KV head waste nothing (rows on the m = 16 side took twice the MMAs and 48
// more registers).  Warp 4 streams pages through a ring of TMA stages; of the other four, warps 0, 1
// take the halves (32 tokens) of even pages and warps 2, 3 of odd ones, each with its own online
// softmax, so the page loop has no CTA barrier.
//
// The pages of all units, laid end to end, are cut into equal ranges, one per CTA of a single wave:
// the lengths are read on the device, so a ragged batch keeps every SM busy to the end.  A unit inside
// one range is finished there; the parts of one that is cut go to a buffer of the call, and a second,
// small kernel joins them in page order.  Nothing is shared between calls, there are no atomics, and
// results do not change from run to run.
//
// Measured (device time of both kernels): 32 sequences of 2048 tokens, 32/8 heads (136 MB), 32.0 us, of
// which the pages take 27 (5.0 TB/s) and the join 4-5.  No unit is full in the page loop (DRAM at 0.71 of
// the copy rate in a profile of it alone, issue slots 39%, ALU 41%): 15 warps to an SM, at 128 registers,
// wait for pages and for their own chain of load, convert, MMA and softmax.  61 ragged sequences up to
// 8191 tokens, 32/4 heads, 24.5 us, against 72 with a CTA to a unit and 35 with four; the same work takes
// 32 equal sequences 28.5 us with a CTA to a unit: equal shares cost them the join.  One of 200 tokens
// 5.5 us, bound by the chain of launch, lengths, page ids, page and join.
//
// Arithmetic.  Codes become f16 fragments exactly (e4m3 is a subset of f16); q is scaled per row by a
// power of two into f16's range.  The value scale joins the exponent: with s the score in the exp2
// domain and e the exponent of V's scale,
//   P = 2^(s + e - m),   O = sum P v8,   l = sum P 2^-e,   m = running max of s + e - 15,   out = O / l,
// which is softmax(s) V for any m, so parts with other references (a prefix's, whose m is max s) join by
// the same formula.  With m from the pages' own s + e, P reaches 2^15 whatever the scales, which uses f16's
// whole range: P v8 down to 2^-29 of the largest is held to 2^-12 of itself, smaller to 2^-40 of the largest.
// S, m, l and O are fp32.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include "sil/fmha.cuh"
#include "sil/host.h"
#include "sil/kv_fp8.cuh"
#include "sil/mma.cuh"
#include "sil/ptx.cuh"

namespace sil {

void check_kv_fp8(const char* what, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& scales, const at::Device& device);

namespace {

constexpr int kMaxRows = 16;                           // query rows of a tile
constexpr int kStages = 4;                              // even: see the page loop
constexpr int kSideBytes = kKvPage * kKvDim;           // K (or V) of one page and head: 8 KB
constexpr int kStageBytes = 2 * kSideBytes;
constexpr int kScaleBytes = 2 * kKvPage;               // both sides' scales of one page and head
constexpr int kWarps = 4;                              // consumer warps
constexpr int kThreads = (kWarps + 1) * 32;
// A context of up to so many pages is one CTA's work.  That goes by the block table's width, which the
// host knows, not by the lengths: one sequence of 200 tokens takes 5.5 us with 4 columns and 7.8 with 16 to
// 512, 32 of them with 8 KV heads 7.6 and 12.6.
constexpr int kWholePages = 8;
// (Geometric mean over 20 decode cases, 1 to 61 sequences, 1 to 20000 tokens: kMinWork 5, 8, 14: 10.6,
// 10.7, 11.6 us; kUnitCost 1, 3, 6: 11.1, 10.6, 10.6; kWholePages 8, 32: 10.6, 10.6.)
constexpr int kUnitCost = 3;                           // what a unit costs beside its pages, in pages
constexpr int kMinWork = 5;                            // of a CTA's range: less costs more than it spreads

// smem map
constexpr int kOffScales = kStages * kStageBytes;
constexpr int kOffBars = kOffScales + kStages * kScaleBytes;
constexpr int kOffUnit = kOffBars + (2 * kStages + 2) * 8;
constexpr int kOffMl = kOffUnit + 64;                  // (m, l) beside two warps' fragments
constexpr int kOffQ = kOffMl + 2 * 2 * 4 * 16 + 112;   // the unit's queries, then the fragments
static_assert(kOffMl % 16 == 0 && kOffQ % 128 == 0, "16-byte joins, aligned queries");
constexpr int kQBytes = 8 * kKvDim * 2;                // of eight rows
constexpr int kFragBytes = 8 * 32 * 16;                // of eight rows and one warp
constexpr int smem_bytes(int tiles) { return kOffQ + tiles * (kQBytes + 2 * kFragBytes); }
static_assert(3 * (smem_bytes(1) + 1024) <= 233472, "three CTAs of eight rows on an SM");

struct Args {
  const __nv_bfloat16* q;
  long long q_stride;      // elements between consecutive tokens
  __nv_bfloat16* out;
  long long o_stride;
  const int* block_table;
  long long bt_stride;
  const int* seq_lens;     // context length incl. the queries
  const int* cu_q;         // [B + 1] query offsets, or null: one query per sequence
  int num_q;               // rows of q
  int max_q;               // queries of a sequence at most (with cu_q)
  const uint8_t* scales;
  int G, Hkv;
  int num_pages, max_pages;   // of the cache; columns of the block table
  int tokens_per_tile;     // query tokens of a tile
  int tiles;               // row tiles per sequence
  int units;               // sequences * tiles * KV heads
  bool whole;              // one CTA per unit: no unit is cut
  float scale_log2;        // softmax scale * log2(e)
  // A batch that shares a prefix (else null): the whole pages of the first prefix_len[0] tokens are
  // already attended, in part_splits parts of equal numbers of 128-key tiles: O [part, B, Hq, 128] in
  // units of 2^60 and (m, l) [part, B, Hq, 2].  They are left out here and joined in.
  const int* prefix_len;
  const float* part_o;
  const float* part_ml;
  int part_splits;             // 0: the prefix is attended here like the rest
  long long part_rows;         // B * Hq
  // Parts of cut units.  Slot 2 w: the part of CTA w that continues a unit; slot 2 w + 1: the one
  // that begins a unit which goes on in CTA w + 1.  cut_id: the unit, or -1.
  float* cut_o;            // [2 CTAs][rows][128]
  float2* cut_ml;          // [2 CTAs][rows]
  int* cut_id;             // [2 CTAs]
  int* status;
};

// Parts of a prefix of `pages` pages that hold anything.
__device__ __forceinline__ int prefix_parts(const Args& a, int pages) {
  const int tiles = (pages + 1) / 2, per = (tiles + a.part_splits - 1) / a.part_splits;
  return (tiles + per - 1) / per;
}

// What a unit's rows are and see.
struct Tile {
  int first, rows;             // first query (row of q), rows of the tile
  int len, pos0;               // context length, position of the first query
  int shared;                  // pages of the prefix that the sequence shares
  int done, pages;             // those of them that another kernel did, pages after them to attend
};

__device__ __forceinline__ Tile tile_of(const Args& a, int v) {   // v = sequence * tiles + tile
  Tile x;
  const int b = v / a.tiles;
  x.len = min(a.seq_lens[b], a.max_pages * kKvPage);
  const int q_begin = a.cu_q != nullptr ? a.cu_q[b] : b;
  int q_len = a.cu_q != nullptr ? a.cu_q[b + 1] - q_begin : 1;
  // Offsets outside q, or more queries than the launch has tiles for: no queries.
  if (q_begin < 0 || q_len < 0 || q_len > a.num_q - q_begin || q_len > a.max_q) {
    raise_status(a.status, kStatusBadArgument);
    q_len = 0;
  }
  const int prefix = a.prefix_len != nullptr ? a.prefix_len[0] : 0;
  const int token0 = (v - b * a.tiles) * a.tokens_per_tile;
  const int tokens = max(0, min(a.tokens_per_tile, q_len - token0));
  x.first = q_begin + token0;
  x.rows = tokens * a.G;
  x.pos0 = x.len - q_len + token0;
  const int seen = tokens > 0 ? min(x.len, x.pos0 + tokens) : 0;   // keys that its last token sees
  // The prefix counts only for a sequence that is that long.
  x.shared = prefix > 0 && x.len >= prefix ? min(prefix / kKvPage, a.max_pages) : 0;
  x.done = a.part_splits > 0 ? x.shared : 0;
  x.pages = max(0, (max(seen, 0) + kKvPage - 1) / kKvPage - x.done);
  return x;
}

// The four codes of w as f16 pairs (codes 0, 1) and (2, 3); exact.
__device__ __forceinline__ void e4m3_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit elements held one pair per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// log2 of the largest P: f16 ends at 2^16.
constexpr float kTop = 15.f;

// Joins partials (m_i, l_i, o_i) of one row: rescaling factor of a part, 0 where there is none.
__device__ __forceinline__ float part_factor(float m, float M) {
  return m == -INFINITY ? 0.f : ex2_approx(m - M);
}

__device__ __forceinline__ void add_part(float4& acc, const float4& o, float f) {
  acc.x = fmaf(o.x, f, acc.x);
  acc.y = fmaf(o.y, f, acc.y);
  acc.z = fmaf(o.z, f, acc.z);
  acc.w = fmaf(o.w, f, acc.w);
}

__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Where row r of a tile goes.
__device__ __forceinline__ __nv_bfloat16* out_row(const Args& a, int first, int h, int r) {
  const int tok = r / a.G;
  return a.out + (long long)(first + tok) * a.o_stride + (long long)(h * a.G + r - tok * a.G) * kKvDim;
}

__device__ __forceinline__ void store4(__nv_bfloat16* to, const float4& o, float f) {
  *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
}

// Tiles without pages of their own: zeros, or the prefix's part alone.  Also the check that a row's
// prefix pages are those of the first row that shares it, through which it is read.
__device__ __forceinline__ void no_page_tiles(const Args& a, int threads) {
  const int sharing = a.prefix_len != nullptr ? first_sharing(a.seq_lens, a.num_q, a.prefix_len[0], threadIdx.x & 31) : -1;
  const int* first = a.block_table + max(0, sharing) * a.bt_stride;
  for (int v = blockIdx.x; v < a.units / a.Hkv; v += gridDim.x) {
    const Tile x = tile_of(a, v);
    const int b = v / a.tiles;
    if (x.pages == 0) {
      for (int e = threadIdx.x; e < a.Hkv * x.rows * 32; e += threads) {
        const int h = e / (32 * x.rows), r = e / 32 % x.rows, dim = 4 * (e & 31);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float f = 0.f;
        if (x.done > 0) {
          float m = -INFINITY, l = 0.f;
          for (int i = 0; i < prefix_parts(a, x.done); ++i) {
            const long long part = i * a.part_rows + ((long long)b * a.Hkv + h) * a.G + r;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + part * 2);
            const float M = fmaxf(m, ml.x), fo = part_factor(m, M), fp = part_factor(ml.x, M);
            o = make_float4(o.x * fo, o.y * fo, o.z * fo, o.w * fo);
            add_part(o, *reinterpret_cast<const float4*>(a.part_o + part * kKvDim + dim), fp);
            l = fmaf(ml.y, fp, l * fo);
            m = M;
          }
          f = 0x1p60f * inverse(l);
        }
        store4(out_row(a, x.first, h, r) + dim, o, f);
      }
    }
    const int* own = a.block_table + (long long)b * a.bt_stride;
    for (int i = threadIdx.x; i < x.shared; i += threads)
      if (own[i] != first[i]) raise_status(a.status, kStatusBadArgument);
  }
}

// A CTA's range of the work of all units: where it begins and how long it is.  A unit's work is its
// pages and kUnitCost more at its front, for what every unit costs beside its pages.
struct Plan {
  int v, h, at;
  long long left;
};

__device__ __forceinline__ int unit_work(const Args& a, int v) {
  const int pages = tile_of(a, v).pages;
  return pages > 0 ? pages + kUnitCost : 0;
}

__device__ __forceinline__ Plan plan_of(const Args& a, int lane) {
  Plan r{};
  if (a.whole) {
    r.v = blockIdx.x / a.Hkv;
    r.h = blockIdx.x % a.Hkv;
    r.left = unit_work(a, r.v);
    return r;
  }
  const int V = a.units / a.Hkv;
  const int n0 = lane < V ? unit_work(a, lane) : 0;   // most batches need no second look
  long long total = 0;
  for (int base = 0; base < V; base += 32) {
    int n = base == 0 ? n0 : base + lane < V ? unit_work(a, base + lane) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  total *= a.Hkv;
  const long long ctas = max(1LL, min((long long)gridDim.x, total / kMinWork));
  if (blockIdx.x >= ctas) return r;
  const long long lo = total * blockIdx.x / ctas;
  r.left = total * (blockIdx.x + 1) / ctas - lo;
  long long before = 0;
  for (int base = 0; base < V; base += 32) {
    const int n = base == 0 ? n0 : base + lane < V ? unit_work(a, base + lane) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + (long long)upto * a.Hkv > lo);
    if (hit != 0) {
      const int first = __ffs(hit) - 1;
      const int work = __shfl_sync(0xffffffffu, n, first);
      const long long at = lo - before - (long long)(__shfl_sync(0xffffffffu, upto, first) - work) * a.Hkv;
      r.v = base + first;
      r.h = static_cast<int>(at / work);
      r.at = static_cast<int>(at % work);
      return r;
    }
    before += (long long)__shfl_sync(0xffffffffu, upto, 31) * a.Hkv;
  }
  return r;
}

// A unit, or the part of it in the CTA's range, as the producer hands it to the other warps.
struct Unit {
  int v, h;
  int p, count;   // first page (of the tile's own) and how many; count 0: the range is done
  Tile x;
};
static_assert(sizeof(Unit) <= 64, "unit slot");

// Whether every consumer thread says yes.
__device__ __forceinline__ bool consumers_agree(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(yes ? 1u : 0u)
      : "memory");
  return r != 0;
}

// kTiles: groups of eight rows.
template <int kTiles>
__global__ void __launch_bounds__(kThreads, kTiles == 1 ? 3 : 2)
    attn_fp8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const Args args) {
  constexpr int kRows = 8 * kTiles;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t* empty = full + kStages;
  uint64_t* unit_full = empty + kStages;
  uint64_t* unit_empty = unit_full + 1;
  Unit* unit = reinterpret_cast<Unit*>(smem + kOffUnit);

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);   // the two warps that share a page
    }
    mbar_init(unit_full, 1);
    mbar_init(unit_empty, kWarps);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  // The swizzled reads count on pages at multiples of 1024 bytes.
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) raise_status(args.status, kStatusBadArgument);
    return;
  }
  pdl_wait();  // q, the cache and the lengths come from earlier kernels

  if (warp == kWarps) {
    // ---------------------------------------------------------------- producer
    int issued = 0, units = 0;   // pages and units handed over
    bool ok = load_status(args.status) == 0;
    // Hands a unit over with its queries (one copy per token: its heads lie side by side), once the
    // consumers have taken the last one from the slot.
    auto hand_over = [&](const Unit& u) {
      if (lane == 0) {
        if (units > 0) ok = mbar_wait(unit_empty, (units - 1) & 1, args.status, kStatusTimeoutEmpty);
        if (ok) {
          *unit = u;
          const int tokens = u.count > 0 ? u.x.rows / args.G : 0;
          const uint32_t bytes = args.G * kKvDim * 2;
          mbar_arrive_expect_tx(unit_full, tokens * bytes);
          for (int i = 0; i < tokens; ++i)
            bulk_load(smem + kOffQ + i * bytes,
                      args.q + (long long)(u.x.first + i) * args.q_stride + (long long)u.h * args.G * kKvDim,
                      bytes, unit_full);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (ok) ++units;
    };
    const Plan plan = plan_of(args, lane);
    long long left = plan.left;
    for (int v = plan.v, h = plan.h, at = plan.at; left > 0 && ok;) {
      Unit u{v, h, max(0, at - kUnitCost), 0, tile_of(args, v)};
      const int work = u.x.pages > 0 ? static_cast<int>(min(left, (long long)(u.x.pages + kUnitCost - at))) : 0;
      u.count = max(0, at + work - kUnitCost) - u.p;
      if (u.count > 0) hand_over(u);
      const int* bt = args.block_table + (long long)(v / args.tiles) * args.bt_stride + u.x.done + u.p;
      for (int base = 0; base < u.count && ok; base += 32) {
        const int n = min(32, u.count - base);
        const int mine = lane < n ? bt[base + lane] : 0;
        for (int j = 0; j < n && ok; ++j) {
          const int pid = __shfl_sync(0xffffffffu, mine, j);
          const int s = issued % kStages;
          if (static_cast<unsigned>(pid) >= static_cast<unsigned>(args.num_pages)) {
            if (lane == 0) raise_status(args.status, kStatusBadArgument);
            ok = false;
            break;
          }
          if (lane == 0) {
            if (issued >= kStages)
              ok = mbar_wait(&empty[s], ((issued / kStages) - 1) & 1, args.status, kStatusTimeoutEmpty);
            if (ok) {
              const int head = pid * args.Hkv + h;
              mbar_arrive_expect_tx(&full[s], kStageBytes + kScaleBytes);
              tma_load_2d(smem + s * kStageBytes, &tmK, &full[s], 0, head * kKvPage);
              tma_load_2d(smem + s * kStageBytes + kSideBytes, &tmV, &full[s], 0, head * kKvPage);
              bulk_load(smem + kOffScales + s * kScaleBytes,
                        args.scales + (long long)head * kScaleBytes, kScaleBytes, &full[s]);
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (ok) ++issued;
        }
      }
      left -= work;
      at = 0;
      if (++h == args.Hkv) {
        h = 0;
        ++v;   // units without pages are passed over: they have no work
      }
    }
    if (ok) hand_over(Unit{});
    // Every load issued has landed before the CTA gives its shared memory back (the consumers wait for
    // the same phases unless one of their waits gave up).
    if (lane == 0) {
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_drain(&full[i % kStages], (i / kStages) & 1);
      if (units > 0) mbar_drain(unit_full, (units - 1) & 1);
    }
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, t = lane & 3;
  float4* frags = reinterpret_cast<float4*>(smem + kOffQ + kTiles * kQBytes);   // [2][kTiles][8][32 lanes]
  float4* frag_ml = reinterpret_cast<float4*>(smem + kOffMl);                   // [2][2][4]
  if (!args.whole && threadIdx.x == 0)
    args.cut_id[2 * blockIdx.x] = args.cut_id[2 * blockIdx.x + 1] = -1;
  no_page_tiles(args, kWarps * 32);                    // (while the producer makes its plan)
  bool alive = true;
  int page = 0;                                        // of the whole range
  for (int n = 0;; ++n) {
    // All consumers go on together, or none (and warp 0 has read the last unit's fragments).
    alive = alive && mbar_wait(unit_full, n & 1, args.status, kStatusTimeoutFull);
    alive = consumers_agree(alive);
    if (!alive) return;
    const int v = unit->v, h = unit->h, p = unit->p, count = unit->count;
    const Tile x = unit->x;
    if (count == 0) break;
    const int rows = x.rows, len = x.len, p_begin = x.done + p;
    float o[kTiles][8][4];                             // O^T: 16-dim blocks x (dims, rows) fragments
    float m_r[kTiles][2], l_r[kTiles][2];              // rows 2 t, 2 t + 1 of each group
    // Q^T fragments: k-step i of thread t covers dims 32 t + 4 i .. 32 t + 4 i + 3 of row g (and the
    // K fragments the same dims: a product does not mind their order).
    uint32_t qb[kTiles][8][2];
    float row_mul[kTiles][2];
    int limit[kTiles][2];                            // keys that rows 2 t, 2 t + 1 see
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      const int r = 8 * u + g;
      uint32_t w[16];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (r < rows)
          q = *reinterpret_cast<const uint4*>(smem + kOffQ + r * kKvDim * 2 + t * 64 + c * 16);
        w[4 * c] = q.x; w[4 * c + 1] = q.y; w[4 * c + 2] = q.z; w[4 * c + 3] = q.w;
      }
      uint32_t amax = 0;
#pragma unroll
      for (int c = 0; c < 16; ++c)
        amax = max(amax, max((w[c] & 0x7fffu), (w[c] >> 16) & 0x7fffu));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // q 2^(14 - E) in f16: exact down to 2^-28 of the row's largest value.
      const int E = max(-100, min(127, static_cast<int>(amax >> 7) - 127));
      const float f = __uint_as_float(static_cast<uint32_t>(14 - E + 127) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qb[u][i][0] = pack_f16x2(bf16_lo(w[2 * i]) * f, bf16_hi(w[2 * i]) * f);
        qb[u][i][1] = pack_f16x2(bf16_lo(w[2 * i + 1]) * f, bf16_hi(w[2 * i + 1]) * f);
      }
      const float mine = args.scale_log2 * __uint_as_float(static_cast<uint32_t>(E - 14 + 127) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        row_mul[u][j] = __shfl_sync(0xffffffffu, mine, (2 * t + j) * 4);
        limit[u][j] = min(len, x.pos0 + (8 * u + 2 * t + j) / args.G + 1);
        m_r[u][j] = -INFINITY;
        l_r[u][j] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) o[u][c][0] = o[u][c][1] = o[u][c][2] = o[u][c][3] = 0.f;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(unit_empty);
    const int all_see = min(len, x.pos0 + 1);          // every row sees the keys below
    const int half = (warp & 1) * 32;

    // Whose page is whose goes by the ring's count, and the ring is even: a stage then belongs to one pair
    // of warps, which has taken the stage's last page before it waits for the next.  (A wait by phase
    // parity needs that: loads land in any order, so the other pair's page could still be on its way.)
    for (int i = ((page & 1) ^ (warp >> 1)); i < count && alive; i += 2) {
      const int s = (page + i) % kStages;
      alive = __all_sync(0xffffffffu, mbar_wait(&full[s], ((page + i) / kStages) & 1, args.status,
                                                kStatusTimeoutFull));
      if (!alive) break;
      const uint32_t kbase = smem_u32(smem + s * kStageBytes) + half * kKvDim;
      const uint32_t vbase = kbase + kSideBytes;
      const uint8_t* sc8 = smem + kOffScales + s * kScaleBytes + half + g;
      const int tok0 = (p_begin + i) * kKvPage + half;
      // S^T: tokens tok0 + 16 a + (g, g + 8), rows 8 u + (2 t, 2 t + 1).
      float sc[2][kTiles][4];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) sc[a][u][0] = sc[a][u][1] = sc[a][u][2] = sc[a][u][3] = 0.f;
        // Token rows g and g + 8, 16-byte chunks 2 t and 2 t + 1 (swizzled by the row).
        const uint32_t row = kbase + (a * 16 + g) * kKvDim;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w0[4], w1[4];
          const uint32_t at = row + (((2 * t + c) ^ g) << 4);
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w0[0]), "=r"(w0[1]), "=r"(w0[2]), "=r"(w0[3]) : "r"(at));
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w1[0]), "=r"(w1[1]), "=r"(w1[2]), "=r"(w1[3]) : "r"(at + 8 * kKvDim));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t ka[4];
            e4m3_to_f16(w0[j], ka[0], ka[2]);
            e4m3_to_f16(w1[j], ka[1], ka[3]);
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
              mma_f16_16816(sc[a][u], ka, qb[u][4 * c + j][0], qb[u][4 * c + j][1]);
          }
        }
      }
      // Scores in the exp2 domain plus the exponent of V's scale.
      float inv_v[2][2];                             // 2^-e of tokens g, g + 8
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t kb = sc8[a * 16 + y * 8], vb = sc8[kKvPage + a * 16 + y * 8];
          const float ks = kv_scale_f32<0>(kb);
          const float ve = vb == kKvScaleNan ? __uint_as_float(0x7fffffffu)
                                             : static_cast<float>(static_cast<int>(vb) - 127);
          inv_v[a][y] = __uint_as_float((254u - min(vb, 253u)) << 23);
#pragma unroll
          for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              sc[a][u][2 * y + j] = fmaf(sc[a][u][2 * y + j] * ks, row_mul[u][j], ve);
        }
      const bool edge = tok0 + 32 > all_see;
      if (edge) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (tok0 + a * 16 + y * 8 + g >= limit[u][j]) sc[a][u][2 * y + j] = -INFINITY;
      }
      uint32_t pb[2][kTiles][2];                     // P^T fragments of the two 16-token steps
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        float alpha[2], m_use[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(fmaxf(sc[0][u][j], sc[0][u][2 + j]), fmaxf(sc[1][u][j], sc[1][u][2 + j]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_new = fmaxf(m_r[u][j], mx - kTop);
          m_use[j] = m_new == -INFINITY ? 0.f : m_new;
          alpha[j] = ex2_approx(m_r[u][j] - m_use[j]);
          m_r[u][j] = m_new;
        }
        // Most pages leave the maxima where they were: the rescale is skipped warp-wide.
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
          l_r[u][0] *= alpha[0];
          l_r[u][1] *= alpha[1];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            o[u][c][0] *= alpha[0]; o[u][c][1] *= alpha[1];
            o[u][c][2] *= alpha[0]; o[u][c][3] *= alpha[1];
          }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float p0 = ex2_approx(sc[a][u][2 * y] - m_use[0]);
            const float p1 = ex2_approx(sc[a][u][2 * y + 1] - m_use[1]);
            l_r[u][0] = fmaf(p0, inv_v[a][y], l_r[u][0]);
            l_r[u][1] = fmaf(p1, inv_v[a][y], l_r[u][1]);
            pb[a][u][y] = transpose8x8(pack_f16x2(p0, p1));
          }
      }
      // V as 8 x 8 tiles of 2-byte units, transposed: a register holds two tokens of two dims, and
      // with its middle bytes exchanged the two tokens of one dim and then of the other.
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t vrow = vbase + (a * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * kKvDim;
        // Bytes behind the context may be no numbers (a weight of 0 does not stop a NaN).
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (edge) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tk = tok0 + a * 16 + y * 8 + 2 * t;
            keep[y] = tk >= len ? 0u : tk + 1 >= len ? 0x0000ffffu : 0xffffffffu;
          }
        }
#pragma unroll
        for (int c2 = 0; c2 < 4; ++c2) {
          const uint32_t c = 2 * c2 + (lane >> 4);
          uint32_t w[4];
          ldmatrix_x4_trans(vrow + ((c ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
          if (edge) {
            w[0] &= keep[0]; w[1] &= keep[1]; w[2] &= keep[0]; w[3] &= keep[1];
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t va[4];   // rows g: dims 2 g, rows g + 8: dims 2 g + 1 of the 16-dim block
            e4m3_to_f16(__byte_perm(w[2 * y], 0u, 0x3120), va[0], va[1]);
            e4m3_to_f16(__byte_perm(w[2 * y + 1], 0u, 0x3120), va[2], va[3]);
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
              mma_f16_16816(o[u][2 * c2 + y], va, pb[a][u][0], pb[a][u][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    // The prefix's parts, where there are any (every fourth part each).  Only now: their m is a maximum
    // of s, without V's exponents, and would put a page's P out of f16's range where those are small.
    if (x.done > 0 && p == 0) {
      const int parts = prefix_parts(args, x.done);
      for (int i = warp; i < parts; i += kWarps)
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = 8 * u + 2 * t + j;
            if (r >= rows) continue;
            const long long part =
                i * args.part_rows + ((long long)(v / args.tiles) * args.Hkv + h) * args.G + r;
            const float2 ml = *reinterpret_cast<const float2*>(args.part_ml + part * 2);
            float2 po[8];
#pragma unroll
            for (int c = 0; c < 8; ++c)
              po[c] = *reinterpret_cast<const float2*>(args.part_o + part * kKvDim + 16 * c + 2 * g);
            const float M = fmaxf(m_r[u][j], ml.x);
            const float fo = part_factor(m_r[u][j], M), fp = part_factor(ml.x, M);
            m_r[u][j] = M;
            l_r[u][j] = fmaf(g == 0 ? ml.y : 0.f, fp, l_r[u][j] * fo);   // a row's lanes are summed at the end
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              o[u][c][j] = fmaf(po[c].x, fp * 0x1p60f, o[u][c][j] * fo);
              o[u][c][2 + j] = fmaf(po[c].y, fp * 0x1p60f, o[u][c][2 + j] * fo);
            }
          }
    }
#pragma unroll
    for (int u = 0; u < kTiles; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l_r[u][j] += __shfl_xor_sync(0xffffffffu, l_r[u][j], d);
    // The warps' (m, l, O) join, lane by lane as the fragments lie: 2 and 3 into 0 and 1, 1 into 0.
    auto put = [&](int slot) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        float4* to = frags + (slot * kTiles + u) * 8 * 32 + lane;
#pragma unroll
        for (int c = 0; c < 8; ++c) to[c * 32] = make_float4(o[u][c][0], o[u][c][1], o[u][c][2], o[u][c][3]);
        if (g == 0) frag_ml[(slot * 2 + u) * 4 + t] = make_float4(m_r[u][0], m_r[u][1], l_r[u][0], l_r[u][1]);
      }
    };
    auto take = [&](int slot) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        const float4* from = frags + (slot * kTiles + u) * 8 * 32 + lane;
        const float4 ml = frag_ml[(slot * 2 + u) * 4 + t];
        const float M0 = fmaxf(m_r[u][0], ml.x), M1 = fmaxf(m_r[u][1], ml.y);
        const float a0 = part_factor(m_r[u][0], M0), a1 = part_factor(m_r[u][1], M1);
        const float b0 = part_factor(ml.x, M0), b1 = part_factor(ml.y, M1);
        m_r[u][0] = M0;
        m_r[u][1] = M1;
        l_r[u][0] = fmaf(ml.z, b0, l_r[u][0] * a0);
        l_r[u][1] = fmaf(ml.w, b1, l_r[u][1] * a1);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 f = from[c * 32];
          o[u][c][0] = fmaf(f.x, b0, o[u][c][0] * a0);
          o[u][c][1] = fmaf(f.y, b1, o[u][c][1] * a1);
          o[u][c][2] = fmaf(f.z, b0, o[u][c][2] * a0);
          o[u][c][3] = fmaf(f.w, b1, o[u][c][3] * a1);
        }
      }
    };
    if (warp >= 2) put(warp - 2);
    const bool clean = consumers_agree(alive);
    if (warp < 2) take(warp);
    __syncwarp();   // every lane of warp 1 has read slot 1
    if (warp == 1) put(1);
    named_bar_sync(1, kWarps * 32);
    if (warp == 0) {
      take(1);
      const bool complete = p == 0 && count == x.pages;
      const long long slot = 2LL * blockIdx.x + (p == 0 ? 1 : 0);
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 8 * u + 2 * t + j;
          if (r >= rows) continue;
          if (!complete) {
            float* to = args.cut_o + (slot * kRows + r) * kKvDim + 2 * g;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<float2*>(to + 16 * c) = make_float2(o[u][c][j], o[u][c][2 + j]);
            if (g == 0) args.cut_ml[slot * kRows + r] = make_float2(m_r[u][j], l_r[u][j]);
          } else if (clean) {
            const float inv = inverse(l_r[u][j]);
            __nv_bfloat16* to = out_row(args, x.first, h, r) + 2 * g;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint32_t*>(to + 16 * c) = pack_bf16x2(o[u][c][j] * inv, o[u][c][2 + j] * inv);
          }
        }
      // (The thread that marked both slots as unused.)
      if (!complete && lane == 0) args.cut_id[slot] = v * args.Hkv + h;
    }
    page += count;
  }
}

// Joins the parts of every unit that begins in CTA w and goes on in w + 1, ...: one CTA each, the
// parts of a row dealt out to several warps, each in page order, and those joined in order.
constexpr int kJoinWarps = 16;

template <int kRows>
__global__ void __launch_bounds__(kJoinWarps * 32) join_cuts_kernel(const Args args, int ctas) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float2 sml[kJoinWarps];
  pdl_trigger();
  pdl_wait();
  const int w0 = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Part i lies in slot 2 (w0 + i), the first one in 2 w0 + 1.
  auto slot_of = [&](int i, int r) { return (2LL * (w0 + i) + (i == 0 ? 1 : 0)) * kRows + r; };
  // Everything that a unit in few parts needs is loaded at once, before it is known what of it counts
  // (the buffer has all slots, whether written or not).
  int rows = args.G;   // one query per sequence needs no lookup
  int groups = max(1, kJoinWarps / rows);   // warps per row
  int r = warp / groups, grp = warp % groups;
  const int id = args.cut_id[2 * w0 + 1];
  const int near = w0 + 1 + lane < ctas ? args.cut_id[2 * (w0 + 1 + lane)] : -1;
  const bool early = args.cu_q == nullptr && r < rows && w0 + grp < ctas;
  float2 ml0 = make_float2(-INFINITY, 0.f);
  float4 po0 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (early) {
    ml0 = args.cut_ml[slot_of(grp, r)];
    po0 = *reinterpret_cast<const float4*>(args.cut_o + slot_of(grp, r) * kKvDim + 4 * lane);
  }
  if (id < 0) return;
  int parts = 1;
  while (true) {   // CTAs in a row whose first part continues this unit
    const int w = w0 + parts + lane;
    const int next = parts == 1 ? near : w < ctas ? args.cut_id[2 * w] : -1;
    const unsigned other = ~__ballot_sync(0xffffffffu, next == id);
    const int more = other == 0 ? 32 : __ffs(other) - 1;
    parts += more;
    if (more < 32) break;
  }
  const int v = id / args.Hkv, h = id % args.Hkv;
  int first = v;
  if (args.cu_q != nullptr) {
    const Tile x = tile_of(args, v);
    first = x.first;
    rows = x.rows;
    groups = max(1, kJoinWarps / max(1, rows));
    r = warp / groups;
    grp = warp % groups;
  }
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (early && parts <= groups) {
    if (grp < parts) {
      m = ml0.x;
      l = ml0.y;
      acc = po0;
    }
  } else if (r < rows) {
    const int each = (parts + groups - 1) / groups;
    const int p0 = grp * each, p1 = min(parts, p0 + each);
    for (int q = p0; q < p1; q += 4) {
      float2 ml[4];
      float4 po[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long at = slot_of(min(q + j, p1 - 1), r);
        ml[j] = args.cut_ml[at];
        po[j] = *reinterpret_cast<const float4*>(args.cut_o + at * kKvDim + 4 * lane);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (q + j >= p1) continue;
        const float M = fmaxf(m, ml[j].x), f = part_factor(m, M), fp = part_factor(ml[j].x, M);
        acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
        add_part(acc, po[j], fp);
        l = fmaf(ml[j].y, fp, l * f);
        m = M;
      }
    }
  }
  so[warp][lane] = acc;
  if (lane == 0) sml[warp] = make_float2(m, l);
  __syncthreads();
  if (r < rows && grp == 0) {
    for (int i = 1; i < groups; ++i) {
      const float2 ml = sml[warp + i];
      const float M = fmaxf(m, ml.x), f = part_factor(m, M), fp = part_factor(ml.x, M);
      acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
      add_part(acc, so[warp + i][lane], fp);
      l = fmaf(ml.y, fp, l * f);
      m = M;
    }
    store4(out_row(args, first, h, r) + 4 * lane, acc, inverse(l));
  }
}

CUtensorMap side_map(const at::Tensor& c) {
  const uint64_t rows = (uint64_t)c.size(0) * c.size(1) * kKvPage;
  return make_tmap_2d(c.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, kKvDim, kKvDim, kKvPage,
                      kKvDim, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

// The output tensor of an attention call over q [T, Hq, 128].
at::Tensor attn_fp8_out(const char* what, const at::Tensor& q, const c10::optional<at::Tensor>& out) {
  if (out.has_value()) return *out;
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == kKvDim, what,
              ": q must be bf16 [T, Hq, 128]");
  c10::cuda::CUDAGuard guard(q.device());
  return at::empty({q.size(0), q.size(1) * kKvDim}, q.options());
}

void check_attn_fp8(const char* what, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& out,
                    double scale) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == kKvDim &&
                  q.stride(2) == 1 && q.stride(1) == kKvDim && q.stride(0) % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15u) == 0,
              what, ": q must be bf16 [T, Hq, 128] with contiguous heads and 16-byte aligned rows");
  const int64_t Hq = q.size(1), Hkv = k_cache.size(1);
  TORCH_CHECK(Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kMaxRows, what,
              ": the query heads must be a multiple of the KV heads, at most 16 to one");
  TORCH_CHECK(out.device() == q.device() && out.scalar_type() == at::kBFloat16 && out.dim() == 2 &&
                  out.size(0) == q.size(0) && out.size(1) == Hq * kKvDim && out.stride(1) == 1 &&
                  out.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15u) == 0,
              what, ": out must be bf16 [T, Hq * 128] with 16-byte aligned rows");
  TORCH_CHECK(seq_lens.device() == q.device() && seq_lens.scalar_type() == at::kInt &&
                  seq_lens.dim() == 1 && seq_lens.is_contiguous(),
              what, ": seq_lens must be contiguous int32 [B] beside q");
  TORCH_CHECK(block_table.device() == q.device() && block_table.scalar_type() == at::kInt &&
                  block_table.dim() == 2 && block_table.size(0) == seq_lens.size(0) &&
                  (block_table.stride(1) == 1 || block_table.size(1) <= 1) &&
                  block_table.size(1) < (1LL << 31) / kKvPage,
              what, ": block_table must be int32 [B, pages] with contiguous rows beside q");
  TORCH_CHECK(seq_lens.size(0) <= 65535, what, ": at most 65535 sequences");
  TORCH_CHECK(scale >= 0.0 && scale < 1e15, what, ": scale must be finite and not negative");
}

namespace {

template <int kTiles>
void launch_attn(const at::Tensor& k_cache, const at::Tensor& v_cache, Args& a, int64_t max_pages,
                 const char* what) {
  constexpr int kRows = 8 * kTiles;
  const CUtensorMap tk = side_map(k_cache), tv = side_map(v_cache);
  const int wave = device_sm_count() * (kTiles == 1 ? 3 : 2);   // CTAs that run at once
  // Short contexts: a unit to a CTA, one launch.  Otherwise one wave with equal shares.
  a.whole = max_pages <= kWholePages;
  int ctas = a.units;
  at::Tensor cut;
  if (!a.whole) {
    ctas = static_cast<int>(std::min<int64_t>(wave, (a.units * (max_pages + kUnitCost) + kMinWork - 1) / kMinWork));
    const int64_t slots = 2LL * ctas * kRows;
    cut = at::empty({slots * (kKvDim + 2) + 2LL * ctas}, k_cache.options().dtype(at::kFloat));
    a.cut_o = cut.data_ptr<float>();
    a.cut_ml = reinterpret_cast<float2*>(a.cut_o + slots * kKvDim);
    a.cut_id = reinterpret_cast<int*>(a.cut_o + slots * (kKvDim + 2));
  }
  auto* kern = attn_fp8_kernel<kTiles>;
  constexpr int smem = smem_bytes(kTiles);
  set_smem_limit(reinterpret_cast<const void*>(kern), smem, "cudaFuncSetAttribute(attn_fp8)");
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  launch_pdl(kern, dim3(ctas), dim3(kThreads), smem, stream, what, tk, tv, a);
  if (!a.whole)
    launch_pdl(join_cuts_kernel<kRows>, dim3(ctas), dim3(kJoinWarps * 32), 0, stream, what, a, ctas);
}

}  // namespace

// Decode (cu_q empty: one query per sequence, q [B, Hq, 128]) and short runs of queries (q packed
// [T, Hq, 128]) -> out [T, Hq * 128]; with prefix_len the part_o / part_ml of prefix_attn_fp8 are
// joined in.
void attn_fp8(const char* what, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
              const at::Tensor& scales, const at::Tensor& block_table, const at::Tensor& seq_lens,
              const int* cu_q, int64_t max_q_len, const at::Tensor& out, double scale, const int* prefix_len,
              const float* part_o, const float* part_ml, int part_splits, const at::Tensor& status) {
  const int64_t B = seq_lens.size(0);
  Args a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.o_stride = out.stride(0);
  a.block_table = block_table.data_ptr<int>();
  a.bt_stride = block_table.stride(0);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.cu_q = cu_q;
  a.num_q = static_cast<int>(q.size(0));
  a.max_q = static_cast<int>(max_q_len);
  a.prefix_len = prefix_len;
  a.part_o = part_o;
  a.part_ml = part_ml;
  a.part_splits = part_splits;
  a.part_rows = B * q.size(1);
  a.scales = scales.data_ptr<uint8_t>();
  a.Hkv = static_cast<int>(k_cache.size(1));
  a.G = static_cast<int>(q.size(1)) / a.Hkv;
  a.num_pages = static_cast<int>(k_cache.size(0));
  a.max_pages = static_cast<int>(block_table.size(1));
  // (At least a tile, which looks at the offsets, if there are to be no queries.)
  const int64_t queries = std::max<int64_t>(1, max_q_len);
  const bool narrow = a.G * queries <= 8;   // one group of eight rows holds a sequence's
  a.tokens_per_tile = (narrow ? 8 : kMaxRows) / a.G;
  const int64_t tiles = (queries + a.tokens_per_tile - 1) / a.tokens_per_tile;
  TORCH_CHECK(B * tiles * a.Hkv < (1LL << 31), what, ": too many query tiles");
  a.tiles = static_cast<int>(tiles);
  a.units = static_cast<int>(B * tiles * a.Hkv);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.status = status.data_ptr<int>();
  (narrow ? launch_attn<1> : launch_attn<2>)(k_cache, v_cache, a, a.max_pages, what);
}

// q [B, Hq, 128] -> out [B, Hq * 128] (allocated unless given).
at::Tensor paged_decode_fp8(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                            const at::Tensor& scales, const at::Tensor& block_table,
                            const at::Tensor& seq_lens, const c10::optional<at::Tensor>& out_, double scale,
                            const at::Tensor& status) {
  const char* what = "paged_decode_fp8";
  const at::Tensor out = attn_fp8_out(what, q, out_);
  check_kv_fp8(what, k_cache, v_cache, scales, q.device());
  check_attn_fp8(what, q, k_cache, block_table, seq_lens, out, scale);
  TORCH_CHECK(q.size(0) == seq_lens.size(0), what, ": one query per sequence");
  if (q.size(0) == 0) return out;
  c10::cuda::CUDAGuard guard(q.device());
  attn_fp8(what, q, k_cache, v_cache, scales, block_table, seq_lens, nullptr, 1, out, scale, nullptr,
           nullptr, nullptr, 0, status);
  return out;
}

}  // namespace sil
