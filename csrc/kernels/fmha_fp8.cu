// Attention of many query rows over the e4m3 KV cache on the 5th-generation tensor cores: causal
// prefill of packed sequences, and the shared prefix of a decode batch.  Format: sil/kv_fp8.cuh.
//
// One CTA per (split of the keys, pair of query tiles, KV head, sequence).  A query tile is up to
// 128 rows, a row being a (token, query head) pair of the heads that share the KV head: 128 / G
// tokens of G heads.  All rows of both tiles use every K / V tile the CTA unpacks, whatever G.
// Four warpgroups (512 threads):
//   warp 0        TMA producer: both Q tiles once, then the e4m3 pages (64 tokens, 8 KB, with
//                 their scale bytes) through a ring of four slots, K one tile ahead of V;
//   warp 1        MMA issuer (one thread) and TMEM owner;
//   warps 4..11   softmax and epilogue, one warpgroup per query tile, one row per thread;
//   warps 12..15  unpacking: e4m3 page -> bf16 K / V tile of 128 tokens in the swizzled layout the
//                 tensor cores read, two stages of each.
// Per key tile: S_X = Q_X K^T (128 x 128 x 128), softmax, O_X += P_X V with P in TMEM over S's
// columns; the two query tiles alternate, so the tensor cores work on one while the other's
// softmax runs.  TMEM (512 columns): S_A | S_B | O_A | O_B.
//
// Unpacking is exact: code times power-of-two scale has 4 significant bits.  The tiles hold K and V
// times 2^-60 (one bf16 multiply by 2^(e + 60) after the bit moves), which the softmax scale and the
// final 1 / l undo.  Tokens past the context become zeros, so nothing that a page holds behind the
// last token reaches a product; a token marked not finite gets NaN keys (masked where it is not
// seen) and zero values.  P is rounded to bf16; m, l, S and O are fp32.
//
// Measured: 1000 queries on 31000 tokens, 32/4 heads, 755-780 us (640-660 TFLOP/s); 558 us with the unpacking's
// work left out, so its issue slots are what the other warps miss, and the chain S, softmax, PV of a
// tile bounds the rest (S_X of the next tile overwrites P_X, so it waits for PV_X).  Steps of 64 keys with
// two S buffers avoid that wait but read Q twice as often and took 839 us.
//
// With few rows the keys are split.  Prefill splits them over the CTAs of a thread-block cluster, which
// join their (m, l, O) through distributed shared memory in split order.  The prefix splits them over
// as many CTAs as there are SMs (clusters of 8 leave 28 of 148 SMs idle, of 16 more) and hands the
// parts to the decode kernel, which takes them in while its own pages are on their way.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "sil/fmha.cuh"
#include "sil/host.h"
#include "sil/kv_fp8.cuh"
#include "sil/ptx.cuh"

namespace sil {

void check_kv_fp8(const char* what, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& scales, const at::Device& device);
void check_attn_fp8(const char* what, const at::Tensor& q, const at::Tensor& k_cache,
                    const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& out,
                    double scale);
at::Tensor attn_fp8_out(const char* what, const at::Tensor& q, const c10::optional<at::Tensor>& out);
void attn_fp8(const char* what, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
              const at::Tensor& scales, const at::Tensor& block_table, const at::Tensor& seq_lens,
              const int* cu_q, int64_t max_q_len, const at::Tensor& out, double scale, const int* prefix_len,
              const float* part_o, const float* part_ml, int part_splits, const at::Tensor& status);

namespace {

constexpr int kBM = 128;                       // rows of a query tile
constexpr int kQT = 2;                         // query tiles per CTA
constexpr int kBN = 128;                       // keys per tile: two pages
constexpr int kHalf = 128 * 64 * 2;            // one [128 rows x 64 dims] bf16 half-tile: 16 KB
constexpr int kTile = 2 * kHalf;
constexpr int kPageBytes = kKvPage * kKvDim;   // one page of e4m3 codes: 8 KB
constexpr int kScaleBytes = 2 * kKvPage;
constexpr int kRing = 4;                       // page slots
constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128;               // 65536 / 512
constexpr int kRegsWg0 = 64, kRegsSoftmax = 184, kRegsUnpack = 80;
static_assert(128 * (kRegsWg0 + kQT * kRegsSoftmax + kRegsUnpack) <= kThreads * kLaunchRegs,
              "register split above the launch allocation");
// Query rows up to which the decode kernel takes a call instead (20 rows on 1500 tokens, 8 sequences,
// 32/8 heads: 16 us against 24 here).
constexpr int kShortRows = 32;
// Pages (of sequences and KV heads, by the block table's width) up to which a shared prefix is not
// attended apart: reading 8192 takes some 33 us, 12 sequences of 6400 tokens and 8 KV heads (9700
// pages) with the prefix apart 37 us.  Contexts much shorter than their table lose by it: 32 sequences on
// 64 shared tokens and 136 own, 8 KV heads, take 22.8 us apart (64 columns) and 12.5 row by row, on 2048
// shared ones 26.7 and 26.5.
constexpr int64_t kUnsharedPages = 8192;
constexpr int kTmemCols = 512;
constexpr uint32_t kColO = 256;                // O_X at kColO + 128 X; S_X / P_X at 128 X

// smem map (offsets from the 1024-aligned base)
constexpr int kOffQ = 0;
constexpr int kOffK = kOffQ + kQT * kTile;     // 2 stages
constexpr int kOffV = kOffK + 2 * kTile;       // 2 stages
constexpr int kOffRing = kOffV + 2 * kTile;
constexpr int kOffScales = kOffRing + kRing * kPageBytes;
constexpr int kOffBar = kOffScales + kRing * kScaleBytes;
constexpr int kSmemBytes = kOffBar + 256 + 1024;
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");
// The join of the splits reuses Q, K and V: O rows padded to 132 floats (a multiple of four banks
// apart, so 16-byte stores of consecutive rows do not collide), then m and l.
constexpr int kJoinLd = kKvDim + 4;
constexpr int kOffJoinM = kQT * kBM * kJoinLd * 4;
constexpr int kOffJoinL = kOffJoinM + kQT * kBM * 4;
static_assert(kOffJoinL + kQT * kBM * 4 <= kOffRing, "the join fits beside the ring");

// A running max may lag the true one by up to 2^8 before O is rescaled (P stays below 256).
constexpr float kRescaleThreshold = 8.0f;

struct Args {
  __nv_bfloat16* out;      // direct output, or null: partial output below
  long long o_stride;
  float* part_o;           // [splits, T, Hq, 128]: O in units of 2^60 and (m, l) of each row, m in the
  float* part_ml;          // [splits, T, Hq, 2]   exp2 domain
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* scales;
  const int* block_table;
  long long bt_stride;
  const int* seq_lens;     // context length incl. the queries
  const int* cu_q;         // [B + 1]; null: one sequence of num_q queries that all see the prefix
  const int* prefix_len;   // [1] tokens, with cu_q null: its whole pages are the keys
  int num_q;               // rows of q
  int max_q;               // queries of a sequence at most (with cu_q)
  int G, Hkv, Hq;
  int num_pages, max_pages;   // of the cache; columns of the block table
  int tokens_per_tile;     // 128 / G
  int splits;
  float scale_log2;        // softmax scale * log2(e) * 2^60
  int* status;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ float4 ld_cluster4(const void* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster1(const void* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// K-major A/B with 128 rows per dim half (1024-byte 8-row atoms stacked along M/N).
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t base, int kslice) {
  return umma_desc_sw128(base + (kslice >> 2) * kHalf + (kslice & 3) * 32);
}

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* status) {
  return mbar_wait(bar, parity, status, kStatusTimeoutFull);
}

// The four codes of w as two bf16 pairs times `mul`: the bf16 words' high bytes (sign, exponent bits
// 7..1) and low bytes (exponent bit 0, mantissa) are made four at a time and interleaved.
__device__ __forceinline__ void unpack4(uint32_t w, uint32_t mul, uint32_t& lo, uint32_t& hi) {
  const uint32_t high = (w & 0x80808080u) | ((w >> 4) & 0x07070707u);
  const uint32_t low = (w << 4) & 0xf0f0f0f0u;
  lo = mul_bf16x2(__byte_perm(low, high, 0x5140), mul);
  hi = mul_bf16x2(__byte_perm(low, high, 0x7362), mul);
}

// kPrefill: causal, packed sequences; else the shared prefix.  (Two instances also because prefill's
// lengths are then uniform to the compiler: with the prefix's row search in the same code 31000 keys
// took 893 us, without it 754 us.)
template <bool kPrefill>
__global__ void __launch_bounds__(kThreads, 1)
    fmha_fp8_kernel(const __grid_constant__ CUtensorMap tmQ, const Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* q_full = bars + 0;
  uint64_t* raw_full = bars + 1;             // [kRing]
  uint64_t* raw_empty = bars + 1 + kRing;    // [kRing], one arrival per unpacking warp
  uint64_t* k_full = bars + 1 + 2 * kRing;   // [2], one arrival per unpacking warp
  uint64_t* k_empty = k_full + 2;            // [2]
  uint64_t* v_full = k_full + 4;             // [2]
  uint64_t* v_empty = k_full + 6;            // [2]
  uint64_t* s_full = k_full + 8;             // [kQT]: S_X in TMEM
  uint64_t* p_full = s_full + kQT;           // [kQT]: P_X in TMEM (128 arrivals)
  uint64_t* o_done = p_full + kQT;           // [kQT]: PV_X finished
  uint64_t* mma_done = o_done + kQT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  int* sflag = reinterpret_cast<int*>(mma_done + 2);   // [0] pages issued

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = args.splits;
  const int split = blockIdx.x % S, pair = gridDim.x / S - 1 - blockIdx.x / S;  // longest first
  const int h = blockIdx.y, b = blockIdx.z;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
    }
    for (int x = 0; x < kQT; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 128);
      mbar_init(&o_done[x], 1);
    }
    mbar_init(mma_done, 1);
    fence_mbar_init();
    sflag[0] = 0;
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  pdl_wait();  // q, the cache and the lengths come from earlier kernels
  const int q_begin = kPrefill ? args.cu_q[b] : 0;
  const int asked = kPrefill ? args.cu_q[b + 1] - q_begin : args.num_q;
  const bool inside = q_begin >= 0 && asked >= 0 && asked <= args.num_q - q_begin && asked <= args.max_q;
  const int q_len = inside ? asked : 0;   // offsets outside q, or too many: no queries (and the status, below)
  // The row of the block table, and the tokens that count.
  int table_row = b, kv_len = 0;
  if constexpr (kPrefill) {
    kv_len = min(args.seq_lens[b], args.max_pages * kKvPage);
  } else {
    table_row = first_sharing(args.seq_lens, args.num_q, args.prefix_len[0], lane);
    if (table_row >= 0) kv_len = max(0, min(args.prefix_len[0] / kKvPage, args.max_pages)) * kKvPage;
  }
  const int pos0 = kv_len - q_len;
  const int tpt = args.tokens_per_tile;
  const int token0 = pair * kQT * tpt;        // first token of tile A; tile X starts X * tpt later
  const bool active = token0 < q_len && load_status(args.status) == 0;
  // Key tiles of query tile X, of the CTA (its split), and of X within the CTA's range.
  int n_x[kQT], n_all = 0;
#pragma unroll
  for (int x = 0; x < kQT; ++x) {
    const int tx = token0 + x * tpt;
    int keys = 0;
    if (active && tx < q_len) keys = kPrefill ? min(pos0 + min(tx + tpt, q_len), kv_len) : kv_len;
    n_x[x] = keys > 0 ? (keys + kBN - 1) / kBN : 0;
    n_all = max(n_all, n_x[x]);
  }
  const int per = (n_all + S - 1) / S;
  const int j0 = split * per;
  int n_tiles = 0;
#pragma unroll
  for (int x = 0; x < kQT; ++x) {
    n_x[x] = max(0, min(n_x[x] - j0, per));
    n_tiles = max(n_tiles, n_x[x]);
  }
  const int n_pages = (kv_len + kKvPage - 1) / kKvPage - 2 * j0;   // pages from the CTA's first tile on
  const int* bt = args.block_table + (long long)table_row * args.bt_stride + 2 * j0;
  const uint32_t sbase = smem_u32(smem);
  const bool joined = kPrefill && S > 1;   // the epilogue goes through shared memory

  // Each setmaxnreg sits inside its own role branch: ptxas compiles the code it dominates with
  // that register budget, so no softmax code may be reachable after the decrease.
  if (warp < 4) {
    regs_dec<kRegsWg0>();
    if (warp == 0) {
      if (lane == 0 && n_tiles > 0) {
        // Q: [G heads x tokens] boxes of 64 dims.  Tokens past the end of q read as zeros, tokens of
        // the next sequence and rows past the box are whatever they are: no such row is stored.
        mbar_arrive_expect_tx(q_full, kQT * 2 * 128 * args.G * tpt);
        for (int x = 0; x < kQT; ++x)
          for (int d = 0; d < 2; ++d)
            tma_load_3d(smem + kOffQ + x * kTile + d * kHalf, &tmQ, q_full, d * 64, h * args.G,
                        q_begin + token0 + x * tpt);
        int issued = 0;
        // Pages 2 i, 2 i + 1 of tile i through the ring; a page past the context is left out.
        auto load_tile = [&](const uint8_t* side, const int (&pg)[2], int i) -> bool {
          for (int p = 0; p < 2; ++p) {
            if (2 * i + p >= n_pages) continue;
            if (static_cast<unsigned>(pg[p]) >= static_cast<unsigned>(args.num_pages)) {
              raise_status(args.status, kStatusBadArgument);
              return false;
            }
            const int s = issued % kRing;
            if (issued >= kRing && !wait_bar(&raw_empty[s], ((issued / kRing) - 1) & 1, args.status))
              return false;
            const long long head = (long long)pg[p] * args.Hkv + h;
            mbar_arrive_expect_tx(&raw_full[s], kPageBytes + kScaleBytes);
            bulk_load(smem + kOffRing + s * kPageBytes, side + head * kPageBytes, kPageBytes, &raw_full[s]);
            bulk_load(smem + kOffScales + s * kScaleBytes, args.scales + head * kScaleBytes, kScaleBytes,
                      &raw_full[s]);
            ++issued;
          }
          return true;
        };
        // Page ids are read one tile before they are used.
        int cur[2] = {0, 0}, prev[2] = {0, 0}, next[2] = {0, 0};
        for (int p = 0; p < 2; ++p) next[p] = p < n_pages ? bt[p] : 0;
        bool ok = true;
        for (int i = 0; i <= n_tiles && ok; ++i) {
          for (int p = 0; p < 2; ++p) {
            prev[p] = cur[p];
            cur[p] = next[p];
            next[p] = (i + 1 < n_tiles && 2 * (i + 1) + p < n_pages) ? bt[2 * (i + 1) + p] : 0;
          }
          if (i < n_tiles) ok = load_tile(args.k, cur, i);
          if (ok && i >= 1) ok = load_tile(args.v, prev, i - 1);
        }
        sflag[0] = issued;
      }
    } else if (warp == 1) {
      if (lane == 0 && n_tiles > 0) {
        const uint32_t idesc_s = umma_idesc_bf16(kBM, kBN);
        const uint32_t idesc_o = umma_idesc_bf16(kBM, kKvDim) | (1u << 16);  // B (V) MN-major
        auto issue_s = [&](int x, int j) {  // S_X = Q_X K_j^T
          const uint32_t qa = sbase + kOffQ + x * kTile;
          const uint32_t kb = sbase + kOffK + (j & 1) * kTile;
#pragma unroll
          for (int k = 0; k < kKvDim / 16; ++k)
            umma_f16(tmem + x * 128, kmajor_desc(qa, k), kmajor_desc(kb, k), idesc_s, k > 0 ? 1u : 0u);
          umma_commit(&s_full[x]);
        };
        auto issue_pv = [&](int x, int j) {  // O_X += P_X V_j, 16 keys (8 TMEM columns) per MMA
          const uint32_t vb = sbase + kOffV + (j & 1) * kTile;
#pragma unroll
          for (int k = 0; k < kBN / 16; ++k)
            umma_f16_ts(tmem + kColO + x * 128, tmem + x * 128 + k * 8,
                        umma_desc_sw128_mn(vb + k * 2048, kHalf), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit(&o_done[x]);
        };
        bool ok = wait_bar(q_full, 0, args.status) && wait_bar(&k_full[0], 0, args.status);
        if (ok) {
          tc_fence_after();
          for (int x = 0; x < kQT; ++x)
            if (n_x[x] > 0) issue_s(x, 0);
          umma_commit(&k_empty[0]);
        }
        for (int j = 0; j < n_tiles && ok; ++j) {
          const int s = j & 1;
          bool v_ready = false, k_ready = false;
          for (int x = 0; x < kQT && ok; ++x) {
            if (j >= n_x[x]) continue;
            if (!wait_bar(&p_full[x], j & 1, args.status)) { ok = false; break; }
            if (!v_ready && !wait_bar(&v_full[s], (j >> 1) & 1, args.status)) { ok = false; break; }
            v_ready = true;
            tc_fence_after();
            issue_pv(x, j);
            if (j + 1 < n_x[x]) {
              // S_X(j+1) overwrites P_X(j), and MMAs with different accumulators are not ordered
              // by the hardware: PV_X(j) must have read it.
              if (!wait_bar(&o_done[x], j & 1, args.status)) { ok = false; break; }
              if (!k_ready && !wait_bar(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, args.status)) {
                ok = false;
                break;
              }
              k_ready = true;
              tc_fence_after();
              issue_s(x, j + 1);
            }
          }
          if (!ok) break;
          umma_commit(&v_empty[s]);
          if (j + 1 < n_tiles) umma_commit(&k_empty[(j + 1) & 1]);
        }
        // Every MMA this thread issued has finished before TMEM is released or the operands'
        // shared memory is used again (also when a wait above gave up).
        umma_commit(mma_done);
        mbar_drain(mma_done, 0);
      }
    }
  } else if (warp < 12) {
    regs_inc<kRegsSoftmax>();
    const int x = (warp - 4) >> 2;          // query tile of this warpgroup
    const int q4 = warp & 3;                // TMEM lane quarter this warp may access
    const int row = q4 * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(q4 * 32) << 16;
    const int n = n_x[x];
    const int tx = token0 + x * tpt;
    const int tok = tx + row / args.G;      // token of this row, and its query head
    const int hq = h * args.G + row % args.G;
    const bool exists = row < tpt * args.G && tok < q_len && active;
    const int limit = kPrefill ? min(kv_len, pos0 + tok + 1) : kv_len;   // keys this row sees
    const int all_see = kPrefill ? min(kv_len, pos0 + tx + 1) : kv_len;  // and every row of the tile
    const uint32_t tS = tmem + x * 128 + lane_off;
    const uint32_t tO = tmem + kColO + x * 128 + lane_off;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // tcgen05.ld / st are warp-collective (.sync.aligned): every branch around them below is made
    // uniform across the warp (__all_sync / __any_sync).
    for (int j = 0; j < n && ok; ++j) {
      ok = __all_sync(0xffffffffu, wait_bar(&s_full[x], j & 1, args.status));
      if (!ok) break;
      tc_fence_after();
      float sv[kBN];
      {
        uint32_t r[kBN];
        tmem_ld64x2_sync(tS, r);
#pragma unroll
        for (int t = 0; t < kBN; ++t) sv[t] = __uint_as_float(r[t]);
      }
      const int key0 = (j0 + j) * kBN;
      if (key0 + kBN > all_see) {
#pragma unroll
        for (int t = 0; t < kBN; ++t)
          if (key0 + t >= limit) sv[t] = -INFINITY;
      }
      float mxp[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) mxp[u] = fmaxf(sv[2 * u], sv[2 * u + 1]);
#pragma unroll
      for (int t = 16; t < kBN; t += 16)
#pragma unroll
        for (int u = 0; u < 8; ++u) mxp[u] = max3f(mxp[u], sv[t + 2 * u], sv[t + 2 * u + 1]);
      const float mx = max3f(max3f(mxp[0], mxp[1], mxp[2]), max3f(mxp[3], mxp[4], mxp[5]),
                             fmaxf(mxp[6], mxp[7]));
      const float mx_s = mx * args.scale_log2;
      float alpha = 1.f;
      if (m == -INFINITY || mx_s > m + kRescaleThreshold) {
        const float m_new = fmaxf(m, mx_s);
        alpha = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
        m = m_new;
      }
      const float m_use = m == -INFINITY ? 0.f : m;
      const uint64_t sc2 = f2(args.scale_log2, args.scale_log2), nm2 = f2(-m_use, -m_use);
      uint64_t acc[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int t = hh * 64 + 2 * c;
          float x0, x1;
          f2_split(fma_f2(f2(sv[t], sv[t + 1]), sc2, nm2), x0, x1);
          const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
          acc[c & 3] = add_f2(acc[c & 3], f2(p0, p1));
          w[c] = pack_bf16x2(p0, p1);
        }
        tmem_st32(tS + hh * 32, w);
      }
      float rsl[4], rsh[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f2_split(acc[u], rsl[u], rsh[u]);
      const float rs = ((rsl[0] + rsh[0]) + (rsl[1] + rsh[1])) + ((rsl[2] + rsh[2]) + (rsl[3] + rsh[3]));
      l = l * alpha + rs;
      if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < kKvDim / 32; ++c) {
          uint32_t r[32];
          tmem_ld32_sync(tO + c * 32, r);
#pragma unroll
          for (int t = 0; t < 32; ++t) r[t] = __float_as_uint(__uint_as_float(r[t]) * alpha);
          tmem_st32(tO + c * 32, r);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }
    // The join reuses the operands' shared memory, so it waits for both tiles' MMAs.
    bool done = ok;
    if (done && n > 0) done = wait_bar(&o_done[x], (n - 1) & 1, args.status);
    if (done && joined && n_tiles > 0) done = wait_bar(mma_done, 0, args.status);
    done = __all_sync(0xffffffffu, done);
    if constexpr (!kPrefill) {
      // A part of the prefix; splits without keys write nothing, and nobody reads them.
      if (done && n > 0) {
        tc_fence_after();
        const long long at = ((long long)split * args.num_q + tok) * args.Hq + hq;
        if (exists) *reinterpret_cast<float2*>(args.part_ml + at * 2) = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < kKvDim / 32; ++c) {
          uint32_t r[32];
          tmem_ld32_sync(tO + c * 32, r);
          if (exists) {
#pragma unroll
            for (int t = 0; t < 32; t += 4)
              *reinterpret_cast<uint4*>(args.part_o + at * kKvDim + c * 32 + t) =
                  make_uint4(r[t], r[t + 1], r[t + 2], r[t + 3]);
          }
        }
      }
    } else if (!joined) {
      if (done) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 0x1p60f / l;
        __nv_bfloat16* orow =
            args.out + (long long)(q_begin + tok) * args.o_stride + (long long)hq * kKvDim;
#pragma unroll 1
        for (int c = 0; c < kKvDim / 32; ++c) {
          uint32_t r[32];
          if (n > 0) {
            tmem_ld32_sync(tO + c * 32, r);
          } else {   // no key is seen: zeros
#pragma unroll
            for (int t = 0; t < 32; ++t) r[t] = 0u;
          }
          if (exists) {
#pragma unroll
            for (int t = 0; t < 32; t += 8) {
              uint4 v;
              v.x = pack_bf16x2(__uint_as_float(r[t + 0]) * inv, __uint_as_float(r[t + 1]) * inv);
              v.y = pack_bf16x2(__uint_as_float(r[t + 2]) * inv, __uint_as_float(r[t + 3]) * inv);
              v.z = pack_bf16x2(__uint_as_float(r[t + 4]) * inv, __uint_as_float(r[t + 5]) * inv);
              v.w = pack_bf16x2(__uint_as_float(r[t + 6]) * inv, __uint_as_float(r[t + 7]) * inv);
              *reinterpret_cast<uint4*>(orow + c * 32 + t) = v;
            }
          }
        }
      }
    } else {
      float* jo = reinterpret_cast<float*>(smem);
      float* jm = reinterpret_cast<float*>(smem + kOffJoinM);
      float* jl = reinterpret_cast<float*>(smem + kOffJoinL);
      tc_fence_after();
      float* mine = jo + (x * kBM + row) * kJoinLd;
      if (done && n > 0) {
#pragma unroll 1
        for (int c = 0; c < kKvDim / 32; ++c) {
          uint32_t r[32];
          tmem_ld32_sync(tO + c * 32, r);
#pragma unroll
          for (int t = 0; t < 32; t += 4)
            *reinterpret_cast<uint4*>(mine + c * 32 + t) = make_uint4(r[t], r[t + 1], r[t + 2], r[t + 3]);
        }
      } else if (n == 0) {
        for (int c = 0; c < kKvDim; c += 4)
          *reinterpret_cast<float4*>(mine + c) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      jm[x * kBM + row] = m;
      jl[x * kBM + row] = l;
      cluster_sync();
      // One row per warp: every CTA of the cluster finishes its share of the rows.
      for (int rr = split * 8 + warp - 4; rr < kQT * kBM; rr += S * 8) {
        const int r = rr % kBM, rt = token0 + rr / kBM * tpt + r / args.G;
        if (r >= tpt * args.G || rt >= q_len || !active) continue;
        float M = -INFINITY;
        for (int sp = 0; sp < S; ++sp) M = fmaxf(M, ld_cluster1(jm + rr, sp));
        const float Mu = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int sp = 0; sp < S; ++sp) {
          const float f = ex2_approx(ld_cluster1(jm + rr, sp) - Mu);
          const float4 v = ld_cluster4(jo + rr * kJoinLd + 4 * lane, sp);
          L += ld_cluster1(jl + rr, sp) * f;
          o.x += v.x * f;
          o.y += v.y * f;
          o.z += v.z * f;
          o.w += v.w * f;
        }
        const int rq = h * args.G + r % args.G;
        const float inv = L == 0.f ? 0.f : 0x1p60f / L;
        *reinterpret_cast<uint2*>(args.out + (long long)(q_begin + rt) * args.o_stride + (long long)rq * kKvDim +
                                  4 * lane) =
            make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
      }
      cluster_sync();  // no CTA leaves while another reads its shared memory
    }
  } else {
    regs_dec<kRegsUnpack>();
    const int tid = threadIdx.x - 384;
    int used = 0;   // pages taken from the ring
    bool ok = true;
    // Pages 2 i, 2 i + 1 as a bf16 tile [dim half][128 tokens][64 dims] at `dst`.  A thread unpacks
    // 16-dim chunk tid & 3 of both halves of the token rows tid / 4 and tid / 4 + 32; odd rows take
    // the halves in the other order, so the eight lanes of a 16-byte phase (two rows) touch all banks
    // once, on the linear side and on the swizzled one.
    auto unpack = [&](uint8_t* dst, int i, bool is_v) {
      for (int p = 0; p < 2; ++p) {
        const bool there = 2 * i + p < n_pages;
        const int s = used % kRing;
        if (there) {
          ok = __all_sync(0xffffffffu, wait_bar(&raw_full[s], (used / kRing) & 1, args.status));
          if (!ok) return;
        }
        const uint8_t* raw = smem + kOffRing + s * kPageBytes;
        const uint8_t* sc = smem + kOffScales + s * kScaleBytes;
        const int left = kv_len - ((j0 + i) * 2 + p) * kKvPage;   // tokens of the page in the context
        uint4 w[4];
#pragma unroll
        for (int it = 0; it < 4; ++it)
          w[it] = *reinterpret_cast<const uint4*>(raw + ((it >> 1) * 32 + (tid >> 2)) * kKvDim +
                                                  (((tid >> 2) ^ it) & 1) * 64 + (tid & 3) * 16);
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int r = rr * 32 + (tid >> 2);
          const uint32_t kb = sc[r], vb = sc[kKvPage + r];
          uint32_t mul = kv_scale_bf16x2<60>(is_v ? vb : kb);
          if (vb == kKvScaleNan) mul = is_v ? 0u : 0x7fff7fffu;
          if (r >= left) mul = 0u;   // codes are finite however stale the page's rest is
          uint8_t* row = dst + (p * kKvPage + r) * 128;
          const uint32_t c0 = ((2 * (tid & 3)) ^ (r & 7)) << 4;
#pragma unroll
          for (int it = 2 * rr; it < 2 * rr + 2; ++it) {
            uint4 o[2];
            unpack4(w[it].x, mul, o[0].x, o[0].y);
            unpack4(w[it].y, mul, o[0].z, o[0].w);
            unpack4(w[it].z, mul, o[1].x, o[1].y);
            unpack4(w[it].w, mul, o[1].z, o[1].w);
            uint8_t* at = row + (((tid >> 2) ^ it) & 1) * kHalf;
            *reinterpret_cast<uint4*>(at + c0) = o[0];
            *reinterpret_cast<uint4*>(at + (c0 ^ 16)) = o[1];
          }
        }
        if (there) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&raw_empty[s]);
          ++used;
        }
      }
    };
    for (int i = 0; i <= n_tiles && n_tiles > 0 && ok; ++i) {
      if (i < n_tiles) {
        const int s = i & 1;
        if (i >= 2) ok = __all_sync(0xffffffffu, wait_bar(&k_empty[s], ((i >> 1) - 1) & 1, args.status));
        if (!ok) break;
        unpack(smem + kOffK + s * kTile, i, false);
        fence_proxy_async_smem();   // the tensor cores read through the async proxy
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&k_full[s]);
      }
      if (i >= 1 && ok) {
        const int j = i - 1, s = j & 1;
        if (j >= 2) ok = __all_sync(0xffffffffu, wait_bar(&v_empty[s], ((j >> 1) - 1) & 1, args.status));
        if (!ok) break;
        unpack(smem + kOffV + s * kTile, j, true);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&v_full[s]);
      }
    }
  }
  if (joined && (warp < 4 || warp >= 12)) {
    cluster_sync();
    cluster_sync();
  }
  if (!inside && threadIdx.x == 0) raise_status(args.status, kStatusBadArgument);
  // Teardown: a producer that gave up lets its own loads land before the CTA exits.
  __syncthreads();
  if (warp == 0 && lane == 0 && n_tiles > 0 && load_status(args.status) != 0) {
    mbar_drain(q_full, 0);
    const int issued = sflag[0];
    for (int i = max(0, issued - kRing); i < issued; ++i) mbar_drain(&raw_full[i % kRing], (i / kRing) & 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();  // tcgen05.dealloc is warp-collective: lane 0 ran the MMA loop alone
    tmem_dealloc(tmem, kTmemCols);
  }
}

// q [T, Hq, 128] as 3-D (dims, heads, tokens), boxes of 64 dims of `heads` x `tokens` rows.
CUtensorMap q_map(const at::Tensor& q, int heads, int tokens) {
  CUtensorMap map;
  const cuuint64_t dims[3] = {kKvDim, (cuuint64_t)q.size(1), (cuuint64_t)q.size(0)};
  const cuuint64_t strides[2] = {kKvDim * 2, (cuuint64_t)q.stride(0) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
  const cuuint32_t unit[3] = {1, 1, 1};
  const CUresult r = tensor_map_encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q.data_ptr(), dims,
                                          strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("fmha_fp8: cuTensorMapEncodeTiled failed");
  return map;
}

int64_t prefix_splits(int64_t ctas, int64_t max_pages, int64_t most) {
  return std::max<int64_t>(1, std::min<int64_t>({most, max_pages / 4, device_sm_count() / ctas}));
}

int64_t tile_pairs(int64_t max_q, int G) {
  const int64_t tokens = kQT * (kBM / G);
  return (max_q + tokens - 1) / tokens;
}

void launch(const char* what, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
            const at::Tensor& scales, const at::Tensor& block_table, const at::Tensor& seq_lens,
            int64_t max_q, int64_t sequences, double scale, const at::Tensor& status,
            Args& a) {
  a.k = static_cast<const uint8_t*>(k_cache.data_ptr());
  a.v = static_cast<const uint8_t*>(v_cache.data_ptr());
  a.scales = scales.data_ptr<uint8_t>();
  a.block_table = block_table.data_ptr<int>();
  a.bt_stride = block_table.stride(0);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.Hkv = static_cast<int>(k_cache.size(1));
  a.Hq = static_cast<int>(q.size(1));
  a.G = a.Hq / a.Hkv;
  a.num_q = static_cast<int>(q.size(0));
  a.max_q = static_cast<int>(max_q);
  a.num_pages = static_cast<int>(k_cache.size(0));
  a.max_pages = static_cast<int>(block_table.size(1));
  a.tokens_per_tile = kBM / a.G;
  // Not 0 (a plain mean of the values): a masked score of -infinity has to stay one when scaled.
  a.scale_log2 = std::max(static_cast<float>(scale * 1.4426950408889634 * 0x1p60), 1e-30f);
  a.status = status.data_ptr<int>();
  auto* fn = a.out != nullptr ? fmha_fp8_kernel<true> : fmha_fp8_kernel<false>;
  const void* kern = reinterpret_cast<const void*>(fn);
  set_smem_limit(kern, kSmemBytes, "cudaFuncSetAttribute(fmha_fp8)");
  // setmaxnreg.inc waits for registers that the other warpgroups hand back; the split adds up to
  // the launch allocation only if the kernel was compiled with kLaunchRegs registers.
  static const bool regs_ok = [] {
    for (const void* k : {reinterpret_cast<const void*>(fmha_fp8_kernel<true>),
                          reinterpret_cast<const void*>(fmha_fp8_kernel<false>)}) {
      cudaFuncAttributes fa{};
      check_cuda(cudaFuncGetAttributes(&fa, k), "cudaFuncGetAttributes(fmha_fp8)");
      if (fa.numRegs != kLaunchRegs) return false;
    }
    return true;
  }();
  TORCH_CHECK(regs_ok, what, ": the kernel was compiled with another register count");
  const int64_t pairs = tile_pairs(max_q, a.G);
  TORCH_CHECK(pairs < (1LL << 27), what, ": too many query tiles");
  // Splits of the keys: as many as leave every SM a CTA at most (the CTA fills an SM), at least two key
  // tiles each; those of prefill are one cluster, 8 at most.
  const bool cluster = a.out != nullptr;
  const int64_t splits = prefix_splits(pairs * a.Hkv * sequences, a.max_pages, cluster ? 8 : 148);
  a.splits = static_cast<int>(splits);
  const CUtensorMap tq = q_map(q, a.G, a.tokens_per_tile);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * splits), a.Hkv, static_cast<unsigned>(sequences));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster ? static_cast<unsigned>(splits) : 1u;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  check_cuda(cudaLaunchKernelEx(&cfg, fn, tq, a), what);
}

}  // namespace

// q: packed [T, Hq, 128]; cu_q [B + 1]; seq_lens [B] (context after append); out [T, Hq * 128]
// (allocated unless given).
at::Tensor paged_prefill_fp8(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                             const at::Tensor& scales, const at::Tensor& block_table,
                             const at::Tensor& seq_lens, const at::Tensor& cu_q, int64_t max_q_len,
                             const c10::optional<at::Tensor>& out_, double scale, const at::Tensor& status) {
  const char* what = "paged_prefill_fp8";
  const at::Tensor out = attn_fp8_out(what, q, out_);
  check_kv_fp8(what, k_cache, v_cache, scales, q.device());
  check_attn_fp8(what, q, k_cache, block_table, seq_lens, out, scale);
  const int64_t B = seq_lens.size(0), Hkv = k_cache.size(1), G = q.size(1) / Hkv;
  TORCH_CHECK(cu_q.device() == q.device() && cu_q.scalar_type() == at::kInt && cu_q.is_contiguous() &&
                  cu_q.numel() == B + 1,
              what, ": cu_q must be contiguous int32 [B + 1] beside q");
  TORCH_CHECK(max_q_len >= 0 && max_q_len < (1LL << 31), what, ": max_q_len must not be negative");
  if (B == 0 || q.size(0) == 0) return out;
  c10::cuda::CUDAGuard guard(q.device());
  // Runs of up to kShortRows rows of a KV head go through the decode kernel.
  if (max_q_len * G <= kShortRows) {
    attn_fp8(what, q, k_cache, v_cache, scales, block_table, seq_lens, cu_q.data_ptr<int>(), max_q_len, out,
             scale, nullptr, nullptr, nullptr, 0, status);
    return out;
  }
  Args a{};
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.o_stride = out.stride(0);
  a.cu_q = cu_q.data_ptr<int>();
  launch(what, q, k_cache, v_cache, scales, block_table, seq_lens, max_q_len, B, scale, status, a);
  return out;
}

// q [B, Hq, 128] -> out [B, Hq * 128] for a batch that shares its first prefix_len tokens: every query
// against the prefix's whole pages (through the first row that is that long) in one pass of the tcgen05 kernel, then
// each sequence's rest with the decode kernel, which joins the two.
at::Tensor paged_decode_shared_fp8(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                   const at::Tensor& scales, const at::Tensor& block_table,
                                   const at::Tensor& seq_lens, const at::Tensor& prefix_len,
                                   const c10::optional<at::Tensor>& out_, double scale,
                                   const at::Tensor& status) {
  const char* what = "paged_decode_shared_fp8";
  const at::Tensor out = attn_fp8_out(what, q, out_);
  check_kv_fp8(what, k_cache, v_cache, scales, q.device());
  check_attn_fp8(what, q, k_cache, block_table, seq_lens, out, scale);
  const int64_t B = seq_lens.size(0), Hq = q.size(1);
  TORCH_CHECK(q.size(0) == B, what, ": one query per sequence");
  TORCH_CHECK(prefix_len.device() == q.device() && prefix_len.scalar_type() == at::kInt &&
                  prefix_len.numel() == 1,
              what, ": prefix_len must be int32 [1] beside q");
  if (B == 0) return out;
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t Hkv = k_cache.size(1);
  // Where every sequence reading all pages of its table's width takes no longer than the two more launches.
  if (B * Hkv * block_table.size(1) <= kUnsharedPages) {
    attn_fp8(what, q, k_cache, v_cache, scales, block_table, seq_lens, nullptr, 1, out, scale,
             prefix_len.data_ptr<int>(), nullptr, nullptr, 0, status);
    return out;
  }
  const int64_t splits = prefix_splits(tile_pairs(B, static_cast<int>(Hq / Hkv)) * Hkv, block_table.size(1), 148);
  const int64_t rows = splits * B * Hq;
  const at::Tensor part = at::empty({rows * (kKvDim + 2)}, q.options().dtype(at::kFloat));
  Args a{};
  a.part_o = part.data_ptr<float>();
  a.part_ml = a.part_o + rows * kKvDim;
  a.prefix_len = prefix_len.data_ptr<int>();
  launch(what, q, k_cache, v_cache, scales, block_table, seq_lens, B, 1, scale, status, a);
  attn_fp8(what, q, k_cache, v_cache, scales, block_table, seq_lens, nullptr, 1, out, scale, a.prefix_len,
           a.part_o, a.part_ml, static_cast<int>(splits), status);
  return out;
}

}  // namespace sil
