// Writing the e4m3 KV cache (per-head RMSNorm, RoPE and quantisation in one pass) and reading
// rows of it back as bf16.  Format: sil/kv_fp8.cuh.
//
// Between the bf16 inputs and the single rounding of each output queries are fp32: the norm
// x * rsqrt(mean x^2 + eps) * w, the rotation (a, b) -> (a c - b s, b c + a s) of dims d and d + 64.
// A key keeps its remainders beside (rotate_sticky), and its norm's sum and factor are fp64.  Both
// kernels are bound by memory traffic.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "sil/host.h"
#include "sil/kv_fp8.cuh"
#include "sil/ptx.cuh"

namespace sil {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                       // lanes that share one head (16 dims each)
constexpr int kHeadsPerBlock = kThreads / kLanes;

struct WriteArgs {
  const __nv_bfloat16* qkv;
  long long ld;
  __nv_bfloat16* q_out;
  long long ldq;
  const int* positions;
  const int* slots;
  const float* cos_sin;      // [max_pos, 128]
  int max_pos;
  const __nv_bfloat16* q_norm;
  const __nv_bfloat16* k_norm;
  float eps;
  uint8_t* k;
  uint8_t* v;
  uint8_t* scales;
  int num_slots;             // pages * 64
  int units;                 // tokens * groups of heads
  int Hq, Hkv;
  int* status;
};

__device__ __forceinline__ void unpack8(const uint4& q, float (&x)[16], int at) {
  x[at + 0] = bf16_lo(q.x); x[at + 1] = bf16_hi(q.x);
  x[at + 2] = bf16_lo(q.y); x[at + 3] = bf16_hi(q.y);
  x[at + 4] = bf16_lo(q.z); x[at + 5] = bf16_hi(q.z);
  x[at + 6] = bf16_lo(q.w); x[at + 7] = bf16_hi(q.w);
}

__device__ __forceinline__ uint4 pack8(const float (&x)[16], int at) {
  return make_uint4(pack_bf16x2(x[at], x[at + 1]), pack_bf16x2(x[at + 2], x[at + 3]),
                    pack_bf16x2(x[at + 4], x[at + 5]), pack_bf16x2(x[at + 6], x[at + 7]));
}

// (a b - c d) (r_hi + r_lo) rounded to odd: the last bit is set where anything is left over, so that
// rounding it once more, to e4m3, gives what rounding the exact value would (a rounding to nearest
// first could end on a tie that the exact value is not on).  Where the products nearly cancel, or with
// the factor's second half, the remainders come to several units of the product y: they are added to
// it, exactly, before the last bit is looked at.  (Dekker's sum: exact unless `more` is the larger of the
// two, for which s has to be below 2^-22 of its products; such a value of a rotated pair is code 0.)
__device__ __forceinline__ float rotate_sticky(float a, float b, float c, float d, float r_hi, float r_lo) {
  // (Intrinsics: a product contracted into the next sum would not be the one whose error is taken.)
  const float p = __fmul_rn(a, b), q = __fmul_rn(c, d);
  const float s = __fsub_rn(p, q), t = __fsub_rn(s, p);
  const float rest = __fadd_rn(__fsub_rn(__fsub_rn(p, __fsub_rn(s, t)), __fadd_rn(q, t)),
                               __fsub_rn(fmaf(a, b, -p), fmaf(c, d, -q)));
  const float y0 = __fmul_rn(s, r_hi);
  const float more = fmaf(s, r_hi, -y0) + fmaf(s, r_lo, rest * r_hi);
  const float y = __fadd_rn(y0, more), left = __fsub_rn(more, __fsub_rn(y, y0));
  const uint32_t bits = __float_as_uint(y);
  // (No remainder of infinities and NaN: both comparisons are false.)
  if ((bits & 1u) == 0 && y != 0.f && (left > 0.f || left < 0.f))
    return __uint_as_float((left > 0.f) == (y > 0.f) ? bits + 1 : bits - 1);
  return y;
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Eight lanes per head: lane i holds dims 8i..8i+7 and 64+8i..64+8i+7, so both halves of a rotated
// pair are in one lane and every access is 16 (codes: 8) bytes wide.  `mask`: the eight lanes.
__device__ __forceinline__ void quantize_head(const WriteArgs& a, const float (&x)[16], int lane,
                                              unsigned mask, int slot, int kvh, bool is_v, bool store) {
  // Largest magnitude as an integer: the bits of non-negative floats order like the values, and
  // infinities and NaN come out on top.
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) amax = max(amax, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(mask, amax, o));
  if (!store) return;
  const bool finite = amax < 0x7f800000u;
  const int e = kv_scale_exponent(amax);
  const float inv = finite ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : 0.f;
  uint32_t code[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    code[j] = finite ? pack_e4m3(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv,
                                 x[4 * j + 3] * inv)
                     : 0u;
  const long long head = (long long)(slot / kKvPage) * a.Hkv + kvh;
  uint8_t* dst = (is_v ? a.v : a.k) + (head * kKvPage + slot % kKvPage) * kKvDim + 8 * lane;
  *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
  *reinterpret_cast<uint2*>(dst + 64) = make_uint2(code[2], code[3]);
  if (lane == 0)
    a.scales[(head * 2 + is_v) * kKvPage + slot % kKvPage] =
        static_cast<uint8_t>(finite ? e + 127 : kKvScaleNan);
}

// One group of eight lanes takes kPer heads of a token: their loads are in flight together and share
// the token's angles.  Traffic is all that counts, so four CTAs to an SM, at 64 registers: with the 68
// and 108 that one and four heads would like, 16384 tokens of 32/8 heads took 110 and 140 us, with one
// and two heads at 64 they took 94 and 79 us (4000 tokens with norms 29 and 32).  Since the keys'
// remainders are added up before the rounding, two heads take 81 us (4.7 TB/s, 71% of the copy rate).
template <int kPer>
__global__ void __launch_bounds__(kThreads, 4) rope_kv_write_fp8_kernel(const WriteArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & (kLanes - 1);
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const int heads = a.Hq + 2 * a.Hkv, blocks = (heads + kPer - 1) / kPer;
  const int unit = blockIdx.x * kHeadsPerBlock + threadIdx.x / kLanes;
  if (unit >= a.units) return;   // a whole group
  const int tok = unit / blocks, h0 = unit % blocks * kPer;
  const int pos = a.positions[tok], slot = a.slots[tok];
  const __nv_bfloat16* row = a.qkv + (long long)tok * a.ld + h0 * kKvDim + 8 * lane;
  uint4 raw[kPer][2];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (h0 + i < heads) {
      raw[i][0] = *reinterpret_cast<const uint4*>(row + i * kKvDim);
      raw[i][1] = *reinterpret_cast<const uint4*>(row + i * kKvDim + 64);
    }
  // A token with a position or a slot outside is not written at all.
  if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_pos) || slot >= a.num_slots) {
    if (lane == 0) raise_status(a.status, kStatusBadArgument);
    return;
  }
  const bool store = slot >= 0;
  float c[8], s[8];
  if (h0 < a.Hq + a.Hkv) {
    const float* cs = a.cos_sin + (long long)pos * kKvDim + 8 * lane;
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      *reinterpret_cast<float4*>(c + j) = *reinterpret_cast<const float4*>(cs + j);
      *reinterpret_cast<float4*>(s + j) = *reinterpret_cast<const float4*>(cs + 64 + j);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int hh = h0 + i;
    if (hh >= heads) break;
    float x[16];
    unpack8(raw[i][0], x, 0);
    unpack8(raw[i][1], x, 8);
    if (hh >= a.Hq + a.Hkv) {
      quantize_head(a, x, lane, mask, slot, hh - a.Hq - a.Hkv, true, store);
      continue;
    }
    const bool is_q = hh < a.Hq;
    const __nv_bfloat16* nw = is_q ? a.q_norm : a.k_norm;
    float w[16];
    if (nw != nullptr) {
      unpack8(*reinterpret_cast<const uint4*>(nw + 8 * lane), w, 0);
      unpack8(*reinterpret_cast<const uint4*>(nw + 64 + 8 * lane), w, 8);
    }
    if (is_q) {
      if (nw != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float rstd = rsqrtf(ss * (1.f / kKvDim) + a.eps);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = x[j] * rstd * w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[j], hi = x[j + 8];
        x[j] = lo * c[j] - hi * s[j];
        x[j + 8] = hi * c[j] + lo * s[j];
      }
      __nv_bfloat16* o = a.q_out + (long long)tok * a.ldq + hh * kKvDim + 8 * lane;
      *reinterpret_cast<uint4*>(o) = pack8(x, 0);
      *reinterpret_cast<uint4*>(o + 64) = pack8(x, 8);
      continue;
    }
    // A key keeps the remainder of every product, so its codes are those of the exact values: x w is
    // exact (two 8-bit significands), the rotation comes first and the norm's factor last.
    float r_hi = 1.f, r_lo = 0.f;
    if (nw != nullptr) {
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < 16; ++j) ss = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), ss);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const double r = rsqrt(ss * (1.0 / kKvDim) + a.eps);
      r_hi = static_cast<float>(r);
      r_lo = static_cast<float>(r - r_hi);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] *= w[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float lo = x[j], hi = x[j + 8];
      x[j] = rotate_sticky(lo, c[j], hi, s[j], r_hi, r_lo);
      x[j + 8] = rotate_sticky(hi, c[j], -lo, s[j], r_hi, r_lo);
    }
    quantize_head(a, x, lane, mask, slot, hh - a.Hq, false, store);
  }
}

struct ReadArgs {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* scales;
  const int* slots;
  int num_slots;
  __nv_bfloat16* k_out;     // [T, Hkv, 128], token strides ldk / ldv
  __nv_bfloat16* v_out;
  long long ldk, ldv;
  int units;                // tokens * 2 * Hkv
  int Hkv;
  int* status;
};

// 16384 tokens of 8 KV heads: 20 us (5.1 TB/s), bound by memory.
// Eight lanes per (token, side, head): 16 codes in, 16 bf16 out.  A code times its power-of-two
// scale is exact in bf16; the factor 2^(e + 120) goes in two steps since it can pass bf16's range.
__global__ void __launch_bounds__(kThreads) read_kv_fp8_kernel(const ReadArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & (kLanes - 1);
  const int unit = blockIdx.x * kHeadsPerBlock + threadIdx.x / kLanes;
  if (unit >= a.units) return;
  const int tok = unit / (2 * a.Hkv), rest = unit % (2 * a.Hkv);
  const int side = rest / a.Hkv, h = rest % a.Hkv;
  const int slot = a.slots[tok];
  uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= a.num_slots) {
    if (lane == 0) raise_status(a.status, kStatusBadArgument);
    return;
  }
  if (slot >= 0) {
    const long long head = (long long)(slot / kKvPage) * a.Hkv + h;
    const uint4 code = *reinterpret_cast<const uint4*>(
        (side ? a.v : a.k) + (head * kKvPage + slot % kKvPage) * kKvDim + 16 * lane);
    const uint32_t up = kv_scale_bf16x2<60>(a.scales[(head * 2 + side) * kKvPage + slot % kKvPage]);
    const uint32_t base = 0x5d805d80u;  // 2^60 as a bf16 pair
    const uint32_t w[4] = {code.x, code.y, code.z, code.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t even = mul_bf16x2(mul_bf16x2(e4m3_even_pair(w[j]), base), up);
      const uint32_t odd = mul_bf16x2(mul_bf16x2(e4m3_odd_pair(w[j]), base), up);
      o[2 * j] = __byte_perm(even, odd, 0x5410);
      o[2 * j + 1] = __byte_perm(even, odd, 0x7632);
    }
    out[0] = make_uint4(o[0], o[1], o[2], o[3]);
    out[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
  __nv_bfloat16* dst = (side ? a.v_out + (long long)tok * a.ldv : a.k_out + (long long)tok * a.ldk) +
                       h * kKvDim + 16 * lane;
  *reinterpret_cast<uint4*>(dst) = out[0];
  *reinterpret_cast<uint4*>(dst + 8) = out[1];
}

bool aligned16(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

}  // namespace

// Shared by every e4m3 cache kernel: layout, types and devices of the cache tensors.
void check_kv_fp8(const char* what, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& scales, const at::Device& device) {
  for (const at::Tensor* c : {&k, &v})
    TORCH_CHECK(c->is_cuda() && c->device() == device && c->scalar_type() == at::kFloat8_e4m3fn &&
                    c->is_contiguous() && c->dim() == 4 && c->size(2) == kKvPage &&
                    c->size(3) == kKvDim && aligned16(*c),
                what, ": the KV cache must be contiguous e4m3 [pages, Hkv, 64, 128] on ", device);
  TORCH_CHECK(k.size(0) == v.size(0) && k.size(1) == v.size(1), what, ": K and V differ in shape");
  TORCH_CHECK(k.size(0) > 0 && k.size(1) > 0, what, ": the KV cache is empty");
  TORCH_CHECK(scales.device() == device && scales.scalar_type() == at::kByte &&
                  scales.is_contiguous() && scales.dim() == 4 && scales.size(0) == k.size(0) &&
                  scales.size(1) == k.size(1) && scales.size(2) == 2 && scales.size(3) == kKvPage &&
                  aligned16(scales),
              what, ": scales must be contiguous uint8 [pages, Hkv, 2, 64] beside the cache");
  TORCH_CHECK(k.size(0) * k.size(1) * kKvPage < (1LL << 31), what,
              ": the cache has too many rows for 32-bit row indices");
}

void rope_kv_write_fp8(at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& slots,
                       const at::Tensor& cos_sin, const c10::optional<at::Tensor>& q_norm_w,
                       const c10::optional<at::Tensor>& k_norm_w, double eps, at::Tensor& k_cache,
                       at::Tensor& v_cache, at::Tensor& scales, int64_t Hq, int64_t Hkv,
                       const c10::optional<at::Tensor>& q_out, const at::Tensor& status) {
  const char* what = "rope_kv_write_fp8";
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 &&
                  qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 && aligned16(qkv),
              what, ": qkv must be bf16 [T, (Hq + 2 Hkv) * 128] with 16-byte aligned rows");
  TORCH_CHECK(Hq > 0 && Hkv > 0 && qkv.size(1) == (Hq + 2 * Hkv) * kKvDim, what,
              ": qkv must hold Hq + 2 Hkv heads of 128");
  check_kv_fp8(what, k_cache, v_cache, scales, qkv.device());
  TORCH_CHECK(k_cache.size(1) == Hkv, what, ": the cache has other KV heads than qkv");
  const int64_t T = qkv.size(0);
  for (const at::Tensor* t : {&positions, &slots})
    TORCH_CHECK(t->device() == qkv.device() && t->scalar_type() == at::kInt && t->is_contiguous() &&
                    t->numel() == T,
                what, ": positions and slots must be contiguous int32 [T] beside qkv");
  TORCH_CHECK(cos_sin.device() == qkv.device() && cos_sin.scalar_type() == at::kFloat &&
                  cos_sin.dim() == 2 && cos_sin.size(1) == kKvDim && cos_sin.is_contiguous() &&
                  aligned16(cos_sin),
              what, ": cos_sin must be contiguous fp32 [max_pos, 128]");
  for (const c10::optional<at::Tensor>* w : {&q_norm_w, &k_norm_w})
    TORCH_CHECK(!w->has_value() ||
                    ((*w)->device() == qkv.device() && (*w)->scalar_type() == at::kBFloat16 &&
                     (*w)->is_contiguous() && (*w)->numel() == kKvDim && aligned16(**w)),
                what, ": norm weights must be contiguous bf16 [128]");
  const at::Tensor* qo = q_out.has_value() ? &*q_out : &qkv;
  if (q_out.has_value())
    TORCH_CHECK(qo->device() == qkv.device() && qo->scalar_type() == at::kBFloat16 && qo->dim() == 3 &&
                    qo->size(0) == T && qo->size(1) == Hq && qo->size(2) == kKvDim &&
                    qo->stride(2) == 1 && qo->stride(1) == kKvDim && qo->stride(0) % 8 == 0 &&
                    aligned16(*qo),
                what, ": q_out must be bf16 [T, Hq, 128] with contiguous heads and 16-byte aligned rows");
  const int64_t heads = Hq + 2 * Hkv;
  TORCH_CHECK(T * heads < (1LL << 31) - kHeadsPerBlock, what, ": too many rows");
  if (T == 0) return;
  c10::cuda::CUDAGuard guard(qkv.device());
  WriteArgs a{};
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  a.ld = qkv.stride(0);
  a.q_out = reinterpret_cast<__nv_bfloat16*>(qo->data_ptr());
  a.ldq = qo->stride(0);
  a.positions = positions.data_ptr<int>();
  a.slots = slots.data_ptr<int>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.max_pos = static_cast<int>(cos_sin.size(0));
  a.q_norm = q_norm_w.has_value() ? reinterpret_cast<const __nv_bfloat16*>(q_norm_w->data_ptr()) : nullptr;
  a.k_norm = k_norm_w.has_value() ? reinterpret_cast<const __nv_bfloat16*>(k_norm_w->data_ptr()) : nullptr;
  a.eps = static_cast<float>(eps);
  a.k = static_cast<uint8_t*>(k_cache.data_ptr());
  a.v = static_cast<uint8_t*>(v_cache.data_ptr());
  a.scales = scales.data_ptr<uint8_t>();
  a.num_slots = static_cast<int>(k_cache.size(0) * kKvPage);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.status = status.data_ptr<int>();
  // Two heads to a group from some twenty CTAs to every SM's place on; below that more CTAs hide more.
  const bool many = T * heads >= 20LL * 4 * device_sm_count() * kHeadsPerBlock;
  a.units = static_cast<int>(T * (many ? (heads + 1) / 2 : heads));
  launch_pdl(many ? rope_kv_write_fp8_kernel<2> : rope_kv_write_fp8_kernel<1>,
             dim3((a.units + kHeadsPerBlock - 1) / kHeadsPerBlock), dim3(kThreads), 0,
             at::cuda::getCurrentCUDAStream(), "rope_kv_write_fp8 launch", a);
}

// -> (k, v) [T, Hkv, 128] (allocated unless given).
std::tuple<at::Tensor, at::Tensor> read_kv_fp8(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                               const at::Tensor& scales, const at::Tensor& slots,
                                               const c10::optional<at::Tensor>& k_out_,
                                               const c10::optional<at::Tensor>& v_out_,
                                               const at::Tensor& status) {
  const char* what = "read_kv_fp8";
  check_kv_fp8(what, k_cache, v_cache, scales, k_cache.device());
  const int64_t T = slots.numel(), Hkv = k_cache.size(1);
  TORCH_CHECK(slots.device() == k_cache.device() && slots.scalar_type() == at::kInt && slots.is_contiguous(),
              what, ": slots must be contiguous int32 beside the cache");
  c10::cuda::CUDAGuard guard(k_cache.device());
  auto made = [&] { return at::empty({T, Hkv, kKvDim}, k_cache.options().dtype(at::kBFloat16)); };
  const at::Tensor k_out = k_out_.has_value() ? *k_out_ : made();
  const at::Tensor v_out = v_out_.has_value() ? *v_out_ : made();
  for (const at::Tensor* o : {&k_out, &v_out})
    TORCH_CHECK(o->device() == k_cache.device() && o->scalar_type() == at::kBFloat16 && o->dim() == 3 &&
                    o->size(0) == T && o->size(1) == Hkv && o->size(2) == kKvDim && o->stride(2) == 1 &&
                    o->stride(1) == kKvDim && o->stride(0) % 8 == 0 && aligned16(*o),
                what, ": outputs must be bf16 [T, Hkv, 128] with contiguous heads and 16-byte aligned rows");
  TORCH_CHECK(T * 2 * Hkv < (1LL << 31) - kHeadsPerBlock, what, ": too many rows");
  if (T == 0) return {k_out, v_out};
  ReadArgs a{};
  a.k = static_cast<const uint8_t*>(k_cache.data_ptr());
  a.v = static_cast<const uint8_t*>(v_cache.data_ptr());
  a.scales = scales.data_ptr<uint8_t>();
  a.slots = slots.data_ptr<int>();
  a.num_slots = static_cast<int>(k_cache.size(0) * kKvPage);
  a.k_out = reinterpret_cast<__nv_bfloat16*>(k_out.data_ptr());
  a.v_out = reinterpret_cast<__nv_bfloat16*>(v_out.data_ptr());
  a.ldk = k_out.stride(0);
  a.ldv = v_out.stride(0);
  a.units = static_cast<int>(T * 2 * Hkv);
  a.Hkv = static_cast<int>(Hkv);
  a.status = status.data_ptr<int>();
  launch_pdl(read_kv_fp8_kernel, dim3((a.units + kHeadsPerBlock - 1) / kHeadsPerBlock), dim3(kThreads),
             0, at::cuda::getCurrentCUDAStream(), "read_kv_fp8 launch", a);
  return {k_out, v_out};
}

}  // namespace sil
