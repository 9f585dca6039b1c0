// kv4.hip - the KV cache in 4 bits (VLRF_HIP_KV_Q4_0): quantizing rows as they are
// appended, reading them back, and attention over it.
//
// A block is 32 consecutive elements of a head's row: d = f16(m / -8) for the
// element m of largest magnitude (the first of equal ones), codes
// c = clamp((int)(fl(x * r) + 8.5), 0, 15) with r = 1 / f32(d) (0 where d is 0),
// standing for (c - 8) * d: the encoder of vlrf_quantize_q4_0, bit for bit.  A
// block that holds an infinity or a NaN gets a NaN scale and reads back as NaN.
#include "../internal.hpp"
#include "kv4_layout.hpp"

#include <cmath>

namespace vlrf_hip {
namespace {

constexpr float kNegInf = -INFINITY;
constexpr uint32_t kNanF16 = 0x7E00u;

// f16(m / -8), the sign put on by hand: a block of zeros has -0, which the product
// loses where the compiler fuses it into the conversion.
__device__ __forceinline__ uint32_t kv4_scale_bits(float m) {
    return __half_as_ushort(__float2half_rn(fabsf(m) * 0.125f)) | (~(__float_as_uint(m) >> 16) & 0x8000u);
}

__device__ __forceinline__ uint32_t kv4_code(float x, float r) {
#pragma clang fp contract(off)
    const float y = x * r;
    return (uint32_t)min(15, max(0, (int)(y + 8.5f)));   // the conversion of a NaN is 0
}

__device__ __forceinline__ float kv4_inverse(uint32_t d16) {
    const float d = f16_bits_to_f32(d16);
    return d != 0.f ? 1.f / d : 0.f;
}

// One thread a block.
__global__ __launch_bounds__(256) void kv4_append_kernel(uint8_t* kc, uint8_t* vc, uint16_t* ks, uint16_t* vs,
                                                         const float* __restrict__ k, const float* __restrict__ v,
                                                         int n_kv, int D, int max_seq, int T, int pos) {
    const int nb = D / 32;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)T * n_kv * nb;
    if (i >= 2 * n) return;
    const bool isv = i >= n;
    const size_t j = isv ? i - n : i;
    const int b = (int)(j % nb), g = (int)(j / nb % n_kv), t = pos + (int)(j / nb / n_kv);
    const float* x = (isv ? v : k) + 32 * j;
    float e[32], amax = 0.f, m = 0.f;
    bool bad = false;
#pragma unroll
    for (int l = 0; l < 32; ++l) {
        e[l] = x[l];
        bad |= !(fabsf(e[l]) < INFINITY);
        if (fabsf(e[l]) > amax) { amax = fabsf(e[l]); m = e[l]; }
    }
    const uint32_t d16 = bad ? kNanF16 : kv4_scale_bits(m);
    const float r = kv4_inverse(d16);
    (isv ? vs : ks)[g * kv4::head_scales(max_seq, D) + kv4::scale(t, b, D)] = (uint16_t)d16;
    uint8_t* c = (isv ? vc : kc) + g * kv4::head_codes(max_seq, D);
#pragma unroll
    for (int l = 0; l < 16; ++l) {
        const uint8_t byte = (uint8_t)(kv4_code(e[2 * l], r) | kv4_code(e[2 * l + 1], r) << 4);
        c[isv ? kv4::v_byte(t, l, b, D) : kv4::k_word(t, l / 4, b, D) + l % 4] = byte;
    }
}

// One thread a byte of two codes.
__global__ __launch_bounds__(256) void kv4_dequant_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                          const uint16_t* __restrict__ ks,
                                                          const uint16_t* __restrict__ vs, int n_kv, int D, int max_seq,
                                                          int ctx, float* __restrict__ K, float* __restrict__ V) {
    const int pairs = D / 2;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)ctx * n_kv * pairs;
    if (i >= n) return;
    const int p = (int)(i % pairs), g = (int)(i / pairs % n_kv), t = (int)(i / pairs / n_kv), b = p / 16, l = p % 16;
    const size_t cb = g * kv4::head_codes(max_seq, D), sb = g * kv4::head_scales(max_seq, D) + kv4::scale(t, b, D);
    const uint32_t kb = kc[cb + kv4::k_word(t, l / 4, b, D) + l % 4], vb = vc[cb + kv4::v_byte(t, l, b, D)];
    const float kd = f16_bits_to_f32(ks[sb]), vd = f16_bits_to_f32(vs[sb]);
    reinterpret_cast<float2*>(K)[i] = make_float2((float)((int)(kb & 15u) - 8) * kd, (float)((int)(kb >> 4) - 8) * kd);
    reinterpret_cast<float2*>(V)[i] = make_float2((float)((int)(vb & 15u) - 8) * vd, (float)((int)(vb >> 4) - 8) * vd);
}

// One workgroup a query row of one head; its four waves take the keys in turn, lane
// l elements 2l and 2l + 1 (d 64: half of the lanes idle), each wave with its own
// running maximum and sum, merged at the end.
template <int D>
__global__ __launch_bounds__(256) void kv4_attn_row_kernel(const float* __restrict__ q, const uint8_t* __restrict__ kc,
                                                           const uint8_t* __restrict__ vc,
                                                           const uint16_t* __restrict__ ks,
                                                           const uint16_t* __restrict__ vs, int n_heads, int rep,
                                                           int max_seq, int T, int ctx, float scale,
                                                           float* __restrict__ out) {
    __shared__ float wm[4], wl[4], wo[4][D];
    const int h = blockIdx.x % n_heads, t = blockIdx.x / n_heads, g = h / rep;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, p = lane % (D / 2), b = p / 16, l = p % 16;
    const bool on = lane < D / 2;
    const int seen = ctx - T + t + 1;
    const size_t row = ((size_t)t * n_heads + h) * D;
    const float q0 = on ? q[row + 2 * p] : 0.f, q1 = on ? q[row + 2 * p + 1] : 0.f;
    kc += g * kv4::head_codes(max_seq, D);
    vc += g * kv4::head_codes(max_seq, D);
    ks += g * kv4::head_scales(max_seq, D);
    vs += g * kv4::head_scales(max_seq, D);
    float m = kNegInf, sum = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j = w; j < seen; j += 4) {
        const size_t si = kv4::scale(j, b, D);
        const uint32_t kb = kc[kv4::k_word(j, l / 4, b, D) + l % 4], vb = vc[kv4::v_byte(j, l, b, D)];
        const float kd = f16_bits_to_f32(ks[si]), vd = f16_bits_to_f32(vs[si]);
        const float dot = on ? (q0 * (float)((int)(kb & 15u) - 8) + q1 * (float)((int)(kb >> 4) - 8)) * kd : 0.f;
        const float s = wave_sum(dot) * scale, mn = fmaxf(m, s);
        const float c = m == kNegInf ? 0.f : expf(m - mn), e = expf(mn == kNegInf ? s : s - mn);   // a NaN score stays
        sum = sum * c + e;
        o0 = o0 * c + e * ((float)((int)(vb & 15u) - 8) * vd);
        o1 = o1 * c + e * ((float)((int)(vb >> 4) - 8) * vd);
        m = mn;
    }
    if (lane == 0) { wm[w] = m; wl[w] = sum; }
    if (on) { wo[w][2 * p] = o0; wo[w][2 * p + 1] = o1; }
    __syncthreads();
    if (threadIdx.x >= D) return;
    float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3])), S = 0.f, O = 0.f;
    for (int i = 0; i < 4; ++i) {
        if (wm[i] == kNegInf && wl[i] == 0.f) continue;   // a wave without keys
        const float f = wm[i] == kNegInf ? 1.f : expf(wm[i] - M);
        S += f * wl[i];
        O += f * wo[i][threadIdx.x];
    }
    out[row + threadIdx.x] = S == 0.f ? 0.f : O / S;
}

}  // namespace

int launch_kv4_append(hipStream_t s, const KVLayer& L, int n_kv, int d_head, int max_seq, const float* k, const float* v,
                      int T, int pos) {
    VH_ARG(T >= 1 && n_kv >= 1 && d_head >= 32 && d_head % 32 == 0, "kv_append: bad shape");
    VH_ARG(pos >= 0 && T <= max_seq - pos, "kv_append: %d rows at %d beyond max_seq %d", T, pos, max_seq);
    const size_t n = 2 * (size_t)T * n_kv * (d_head / 32);
    VH_LAUNCH(kv4_append_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, reinterpret_cast<uint8_t*>(L.k),
              reinterpret_cast<uint8_t*>(L.v), reinterpret_cast<uint16_t*>(L.ks), reinterpret_cast<uint16_t*>(L.vs), k, v,
              n_kv, d_head, max_seq, T, pos);
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

int launch_kv4_dequant(hipStream_t s, const KVLayer& L, int n_kv, int d_head, int max_seq, int ctx_len, float* K,
                       float* V) {
    VH_ARG(ctx_len >= 1 && ctx_len <= max_seq, "kv_dequant: ctx_len %d outside [0,%d]", ctx_len, max_seq);
    const size_t n = (size_t)ctx_len * n_kv * (d_head / 2);
    VH_LAUNCH(kv4_dequant_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
              reinterpret_cast<const uint8_t*>(L.k), reinterpret_cast<const uint8_t*>(L.v),
              reinterpret_cast<const uint16_t*>(L.ks), reinterpret_cast<const uint16_t*>(L.vs), n_kv, d_head, max_seq,
              ctx_len, K, V);
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

int launch_attn_kv4(hipStream_t s, const float* q, const KVLayer& L, int n_heads, int n_kv, int d_head, int max_seq, int T,
                    int ctx_len, float scale, float* out) {
    VH_ARG(n_kv >= 1 && n_heads >= 1 && n_heads % n_kv == 0, "attn: n_heads %d not a multiple of n_kv %d", n_heads, n_kv);
    VH_ARG(d_head == 64 || d_head == 128, "attn: d_head %d not in {64,128}", d_head);
    VH_ARG(ctx_len >= 1 && ctx_len <= max_seq && T >= 1 && T <= ctx_len, "attn: %d rows of %d keys in a cache of %d", T,
           ctx_len, max_seq);
    const dim3 grid((unsigned)((size_t)T * n_heads));
#define VH_ROW(D)                                                                                                     \
    VH_LAUNCH(kv4_attn_row_kernel<D>, grid, dim3(256), 0, s, q, reinterpret_cast<const uint8_t*>(L.k),                \
              reinterpret_cast<const uint8_t*>(L.v), reinterpret_cast<const uint16_t*>(L.ks),                         \
              reinterpret_cast<const uint16_t*>(L.vs), n_heads, n_heads / n_kv, max_seq, T, ctx_len, scale, out)
    if (d_head == 64) VH_ROW(64);
    else VH_ROW(128);
#undef VH_ROW
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

}  // namespace vlrf_hip
