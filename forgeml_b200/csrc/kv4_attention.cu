// Attention over the 4-bit key/value cache (neb_kv4_attention).
//
//   out[b,t,h,:] = sum_j p_j v_j,  p = softmax_j(scale * q[b,t,h,:] . k_j),
//   j = 0 .. start_pos[b] + t,     k_j, v_j = z + c * s per group (kv4.cuh)
#include <string>

#include "kv4.cuh"

namespace fml {
namespace kv4 {

constexpr int kWarps = 8;

// One CTA per (request, token, query head), a warp per row; lane l holds
// channels 32 g + l.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    attn_kernel(const T* __restrict__ q, long long qs0, long long qs1, long long qs2, const Pool p,
                const int32_t* __restrict__ slot_of, const int32_t* __restrict__ start_pos, T* __restrict__ out,
                int tq, int QH, float scale) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm_o[kWarps][kMaxD], sm_m[kWarps], sm_l[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int qh = blockIdx.x % QH, t = (blockIdx.x / QH) % tq, b = blockIdx.x / QH / tq;
  const int h = qh / (QH / p.H);
  const int slot = slot_of[b], start = start_pos[b];
  const bool bad = slot < 0 || slot >= p.slots || start < 0 || start > p.max_seq - 1 - t;
  T* op = out + (((long long)b * tq + t) * QH + qh) * p.D;
  if (bad) {
    if (threadIdx.x == 0) raise_device_error(DEV_ERR_ATTN_RANGE);
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) op[d] = from_f32<T>(0.f);
    return;
  }
  const long long r0 = head_row(p, slot, h);
  constexpr int MG = kMaxD / kGroup;
  float qv[MG], o[MG];
#pragma unroll
  for (int g = 0; g < MG; ++g) {
    const int c = g * 32 + lane;
    qv[g] = c < p.D ? to_f32<T>(q[b * qs0 + t * qs1 + qh * qs2 + c]) * scale : 0.f;
    o[g] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int pos = warp; pos <= start + t; pos += kWarps) {
    const long long r = r0 + pos;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < MG; ++g) {
      if (g >= p.G) break;
      const int c = g * 32 + lane;
      const T* pr = static_cast<const T*>(p.kp) + (r * p.G + g) * 2;
      const int code = p.kc[r * 16 * p.G + k_byte(p.G, c)] >> (4 * (c & 1)) & 15;
      if (c < p.D) s = fmaf(qv[g], fmaf((float)code, to_f32<T>(pr[0]), to_f32<T>(pr[1])), s);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mn = fmaxf(m, s), alpha = expf(m - mn), pr_ = expf(s - mn);
    l = l * alpha + pr_;
    m = mn;
#pragma unroll
    for (int g = 0; g < MG; ++g) {
      if (g >= p.G) break;
      const int c = g * 32 + lane;
      const T* pr = static_cast<const T*>(p.vp) + (r * p.G + g) * 2;
      const int code = p.vc[r * 16 * p.G + v_byte(p.G, c, pos)] >> (4 * (c & 1)) & 15;
      o[g] = fmaf(pr_, fmaf((float)code, to_f32<T>(pr[0]), to_f32<T>(pr[1])), o[g] * alpha);
    }
  }
#pragma unroll
  for (int g = 0; g < MG; ++g) sm_o[warp][g * 32 + lane] = o[g];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  __syncthreads();
  float mm = -INFINITY, ll = 0.f, w[kWarps];
  for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, sm_m[i]);
  for (int i = 0; i < kWarps; ++i) {
    w[i] = sm_m[i] == -INFINITY ? 0.f : expf(sm_m[i] - mm);
    ll += w[i] * sm_l[i];
  }
  for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
    float acc = 0.f;
    for (int i = 0; i < kWarps; ++i) acc += w[i] * sm_o[i][d];
    op[d] = from_f32<T>(acc / ll);
  }
}

template <typename T>
static int attention(const void* q, const int64_t* qs, const Pool& p, const int32_t* slot_of, const int32_t* start_pos,
                     void* out, int64_t batch, int64_t t, int64_t q_heads, float scale, cudaStream_t st) {
  const cudaError_t e =
      launch_pdl(attn_kernel<T>, dim3((unsigned)(batch * t * q_heads)), dim3(kWarps * 32), 0, st, 1,
                 static_cast<const T*>(q), (long long)qs[0], (long long)qs[1], (long long)qs[2], p, slot_of, start_pos,
                 static_cast<T*>(out), (int)t, (int)q_heads, scale);
  count_launch();
  return check_cuda(e, "neb_kv4_attention launch");
}

}  // namespace kv4
}  // namespace fml

using namespace fml;

extern "C" int neb_kv4_attention(const void* q, const int64_t q_strides[4], const neb_kv4_pool* pool,
                                 const int32_t* slot_of, const int32_t* start_pos, void* out, int64_t batch,
                                 int64_t t, int64_t q_heads, float scale, void* stream) {
  kv4::Pool p;
  if (const int rc = kv4::pool_from(pool, "neb_kv4_attention", &p)) return rc;
  if (!q || !q_strides || !slot_of || !start_pos || !out) return fail(FML_EINVAL, "neb_kv4_attention: null pointer");
  if (batch <= 0 || t <= 0 || q_heads <= 0) return fail(FML_EINVAL, "neb_kv4_attention: sizes must be positive");
  if (q_heads % p.H != 0) return fail(FML_EINVAL, "neb_kv4_attention: q_heads must be a multiple of the pool's heads");
  if (q_strides[3] != 1) return fail(FML_EUNSUPPORTED, "neb_kv4_attention: q innermost stride must be 1");
  if (t > p.max_seq) return fail(FML_EINVAL, "neb_kv4_attention: t exceeds max_seq");
  if (batch > (1 << 24) || q_heads > (1 << 20) || batch * t > (1ll << 31) / q_heads / 8)
    return fail(FML_EUNSUPPORTED, "neb_kv4_attention: too many queries");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == FML_F32)
    return kv4::attention<float>(q, q_strides, p, slot_of, start_pos, out, batch, t, q_heads, scale, st);
  if (pool->dtype == FML_BF16)
    return kv4::attention<__nv_bfloat16>(q, q_strides, p, slot_of, start_pos, out, batch, t, q_heads, scale, st);
  return kv4::attention<__half>(q, q_strides, p, slot_of, start_pos, out, batch, t, q_heads, scale, st);
}
