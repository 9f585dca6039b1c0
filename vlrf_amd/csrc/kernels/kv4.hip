// kv4.hip - the KV cache in 4 bits (VLRF_HIP_KV_Q4_0): quantizing rows as they are
// appended, reading them back, and attention over it.
//
// A block is 32 consecutive elements of a head's row: d = f16(m / -8) for the
// element m of largest magnitude (the first of equal ones), codes
// c = clamp((int)(fl(x * r) + 8.5), 0, 15) with r = 1 / f32(d) (0 where d is 0),
// standing for (c - 8) * d: the encoder of vlrf_quantize_q4_0, bit for bit.  A
// block that holds an infinity or a NaN gets a NaN scale and reads back as NaN.
#include "../internal.hpp"
#include "attn_core.hpp"
#include "kv4_layout.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace vlrf_hip {
namespace {

constexpr float kNegInf = -INFINITY;
constexpr uint32_t kNanF16 = 0x7E00u;
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

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

// Appending.  A workgroup takes CB blocks of 32 elements of one head's K or V rows at a
// group of 32 key positions, a thread eight elements of a row (the heads of a group
// follow each other, so that whole rows are read at a time: 16000 rows of 8 heads of
// 128 29 us, with the groups of a head side by side 32):
// the four lanes of a block find its extreme by quad exchanges, and each has a word of
// codes.  K's words go out as they are, a row's side by side.  V's bytes and the scales
// are turned in LDS, where a whole group's are side by side, and go out in words; of a
// group that the rows fill in part, byte by byte, so that the others stay.
// Bound by the rows' bytes: that is 149 MB at 5.1 TB/s.  One row takes the time of the call.
struct Kv4Append {
    const float *k, *v;       // [T][ld]
    uint8_t *kc, *vc;
    uint16_t *ks, *vs;
    int ld, D, n_kv, max_seq, T, pos;
    const int* pos_dev;       // the position, from the device (T 1); or null
    const float *cos_t, *sin_t;   // [max_seq][D / 2] (ROPE)
};

__device__ __forceinline__ float quad_f(float v, int which) {   // the lane 1 or 2 away within its four
    return which == 1 ? dpp_f<0xB1>(v) : dpp_f<0x4E>(v);
}

// ROPE: K's rows are rotated at their positions first (rope.hpp:75-99), the element half a
// head away read beside the own one.
template <int CB, bool ROPE>
__global__ __launch_bounds__(128 * CB) void kv4_append_kernel(Kv4Append a) {
    __shared__ uint32_t codes[128 * CB];
    __shared__ uint16_t scales[32 * CB];
    const int tid = threadIdx.x, bl = tid % (4 * CB) / 4, word = tid % 4, slot_key = tid / (4 * CB);
    const bool isv = blockIdx.z & 1;
    const int nb = a.D / 32, b = (int)(blockIdx.z >> 1) * CB + bl, g = blockIdx.x % a.n_kv;
    const int pos = a.pos_dev ? *a.pos_dev : a.pos;
    if (pos < 0 || pos > a.max_seq - a.T) return;   // host checks capacity; never write past the cache
    const int kb = pos / kv4::kKeys + (int)blockIdx.x / a.n_kv, t = kb * kv4::kKeys + slot_key, row = t - pos;
    const bool on = row >= 0 && row < a.T;
    const bool whole = kb * kv4::kKeys >= pos && (kb + 1) * kv4::kKeys <= pos + a.T;

    float e[8] = {};
    const float* from = (isv ? a.v : a.k) + (size_t)row * a.ld + g * a.D;
    const int el = 32 * b + 8 * word;
    if (on) __builtin_memcpy(e, from + el, 32);
    if (ROPE && on && !isv) {
        const int half = a.D / 2, j = el < half ? el : el - half;   // half is a multiple of 8
        float o[8], cr[8], sr[8];
        __builtin_memcpy(o, from + (el < half ? el + half : j), 32);
        __builtin_memcpy(cr, a.cos_t + (size_t)t * half + j, 32);
        __builtin_memcpy(sr, a.sin_t + (size_t)t * half + j, 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float y0, y1;
            attn::rope2(el < half ? e[i] : o[i], el < half ? o[i] : e[i], cr[i], sr[i], &y0, &y1);
            e[i] = el < half ? y0 : y1;
        }
    }
    // The largest magnitude, the first of equal ones: the maximum of (|x|, -index, sign).
    float amax = 0.f, m = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bad |= !(fabsf(e[i]) < INFINITY);
        if (fabsf(e[i]) > amax) { amax = fabsf(e[i]); m = e[i]; }
    }
    if (bad) m = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int step = 1; step <= 2; ++step) {
        const float o = quad_f(m, step);
        const bool below = (word & step) != 0;                       // the other lane's elements come first
        if (o != o || fabsf(o) > fabsf(m) || (below && fabsf(o) == fabsf(m))) m = o;   // a NaN m loses no comparison
    }
    const uint32_t d16 = m != m ? kNanF16 : kv4_scale_bits(m);
    const float r = kv4_inverse(d16);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= kv4_code(e[i], r) << (4 * i);

    uint8_t* cs = (isv ? a.vc : a.kc) + g * kv4::head_codes(a.max_seq, a.D);
    uint16_t* ds = (isv ? a.vs : a.ks) + g * kv4::head_scales(a.max_seq, a.D);
    if (!isv && on) *reinterpret_cast<uint32_t*>(cs + kv4::k_word(t, word, b, a.D)) = w;
    if (!whole) {
        if (!on) return;
        if (isv) {
#pragma unroll
            for (int i = 0; i < 4; ++i) cs[kv4::v_byte(t, 4 * word + i, b, a.D)] = (uint8_t)(w >> (8 * i));
        }
        if (word == 0) ds[kv4::scale(t, b, a.D)] = (uint16_t)d16;
        return;
    }
    const int L = kv4::lane_group(t), slot = kv4::slot(t);
    if (isv) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint8_t*>(codes)[8 * ((L * 16 + 4 * word + i) * CB + bl) + slot] = (uint8_t)(w >> (8 * i));
    }
    if (word == 0) scales[8 * (L * CB + bl) + slot] = (uint16_t)d16;
    __syncthreads();
    const int b0 = b - bl, t0 = kb * kv4::kKeys;
    if (isv) {   // word 2 (run * CB + block) + half of the turned codes
        const int run = tid / (2 * CB), blk = tid / 2 % CB;
        *reinterpret_cast<uint32_t*>(cs + kv4::v_byte(t0, 0, 0, a.D) + 8 * (run * nb + b0 + blk) + 4 * (tid & 1)) = codes[tid];
    }
    if (tid < 16 * CB) {
        const int grp = tid / (4 * CB), blk = tid / 4 % CB;
        *reinterpret_cast<uint32_t*>(ds + kv4::scale(t0, 0, a.D) + 8 * (grp * nb + b0 + blk) + 2 * (tid & 3)) =
            reinterpret_cast<const uint32_t*>(scales)[tid];
    }
}

// Reading back.  A workgroup takes CB blocks of one head at a group of 32 keys: of K a
// thread four elements of a row at a time, of V a byte of eight keys, halves exchanged
// between neighbours so that it writes four elements of four keys.  Heads follow each
// other, so that whole rows are written at a time: 30001 rows of 8 heads of 128 43.8 us,
// with the groups of a head side by side 62.  Bound by the bytes: that is 6.4 TB/s.
template <int CB>
__global__ __launch_bounds__(256) void kv4_dequant_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                          const uint16_t* __restrict__ ks,
                                                          const uint16_t* __restrict__ vs, int row, int D, int max_seq,
                                                          int ctx, float* __restrict__ K, float* __restrict__ V) {
    const int nb = D / 32, b0 = blockIdx.z * CB, g = blockIdx.x % (row / D), t0 = blockIdx.x / (row / D) * kv4::kKeys, tid = threadIdx.x;
    const size_t cb = g * kv4::head_codes(max_seq, D), sb = g * kv4::head_scales(max_seq, D);
    // Past the caches (nontemporal): what is written here is far more than they hold, or
    // read once (30001 rows 43.8 us, through them 66.5; 4096 rows of 4 heads of 64 4.5 both).
    auto put = [&](float* to, int t, int e, float4 x) {
        if (t < ctx) __builtin_nontemporal_store(__builtin_bit_cast(f4v, x), reinterpret_cast<f4v*>(to + (size_t)t * row + g * D + e));
    };
    auto value = [](uint32_t w, int i, float d) { return (float)((int)(w >> (4 * i) & 15u) - 8) * d; };
    constexpr int KI = 256 * CB;   // items of K: 32 keys, 8 CB times four elements
#pragma unroll
    for (int m = tid; m < KI; m += 256) {
        const int q = m % (8 * CB), t = t0 + m / (8 * CB), b = b0 + q / 8;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + cb + kv4::k_word(t, q % 8 / 2, b, D)) >> (16 * (q & 1));
        const float d = f16_bits_to_f32(ks[sb + kv4::scale(t, b, D)]);
        put(K, t, 32 * b0 + 4 * q, make_float4(value(w, 0, d), value(w, 1, d), value(w, 2, d), value(w, 3, d)));
    }
    constexpr int VI = 64 * CB;    // items of V: 4 groups of keys, CB blocks, 16 bytes
#pragma unroll
    for (int m = tid; m < VI; m += 256) {
        const int i = m % 16, bl = m / 16 % CB, L = m / (16 * CB), b = b0 + bl;
        uint2 x = *reinterpret_cast<const uint2*>(vc + cb + kv4::v_byte(t0, 0, 0, D) + 8 * ((L * 16 + i) * nb + b));
        const uint4 d = *reinterpret_cast<const uint4*>(vs + sb + kv4::scale(t0, 0, D) + 8 * (L * nb + b));
        // Even lanes take slots 0..3 of both bytes, odd lanes slots 4..7.
        const bool odd = i & 1;
        const uint32_t give = odd ? x.x : x.y, keep = odd ? x.y : x.x;
        const uint32_t got = __float_as_uint(dpp_f<0xB1>(__uint_as_float(give)));
        const uint32_t lo = odd ? got : keep, hi = odd ? keep : got;   // bytes of elements 4 (i / 2) .. + 1 and + 2 .. + 3
        const uint2 dd = odd ? make_uint2(d.z, d.w) : make_uint2(d.x, d.y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t p = lo >> (8 * j), q = hi >> (8 * j);
            const float s = f16_bits_to_f32(((j & 2) ? dd.y : dd.x) >> (16 * (j & 1)) & 0xFFFFu);
            put(V, t0 + kv4::key_of(L, (odd ? 4 : 0) + j), 32 * b + 2 * (i & ~1),
                make_float4(value(p, 0, s), value(p, 1, s), value(q, 0, s), value(q, 1, s)));
        }
    }
}

// ---- attention --------------------------------------------------------------------
// The T * rep query rows of a KV head (rep query heads share it) stand as rows t rep
// + r.  For few of them a workgroup takes 16, and where blocks of 16 are few several
// share a block's keys (for the fewest, as said at "few rows", 16 / NB): the eight or
// four waves of each take groups of 32 keys in turn, each with its own running maximum
// and sum, and merge through LDS, and the workgroup that comes last merges all of a
// block's.
// One decode row at 32/8 heads of 128: 120001 keys 33.9 us (138 MB, 4.1 TB/s: each byte read
// once, a wave with one group of keys in flight waits 39 % of its time and vector
// instructions take half of every SIMD's; a GEMV of this library reads at 5.1 TB/s); 15001
// keys 9.7 (17 MB, 1.8 TB/s) and 1500 keys 6.7, bound by the chain of
// waits: the launch, the arguments, q and the keys, the group's products and weights, the waves'
// merge, the counter, the chunks' merge, 0.3 to 0.9 us each.
//   scores   S^T = K Q^T, 16 keys by 16 rows and a block of 32 elements an
//            instruction.  A code minus 8 is exact in f16; q, scaled by a power of
//            two for the row's largest element to lie in [2^13, 2^14), enters as two
//            f16 pieces (22 bits).  Each block's sum is scaled in f32.
//   weights  p = 2^(s - m + 10).  m moves when a score passes it by 4 (in powers of
//            two), so p <= 2^14; rescaling O is rare and skipped by the wave.
//   output   O^T = V^T P^T over the same codes: p times the key's scale, in two f16
//            pieces, is the other operand.  With scales from 2^-11 to below 2 (or 0) it
//            stays below 2^15, and the second piece, which rounds at 2^-25 at the
//            finest, is off by 2^-24 at most of the largest weight (2^10 or more) times the
//            scale.  Groups of 32 keys with another scale have their products formed
//            apart, each row's times the power of two that brings the largest that
//            the row sees to [2^14, 2^15), and added scaled back: no key's scale costs
//            another's bits, and a key that the row does not see has no say.  Where
//            every group goes that way (values of 1e-3, or of 1e4) a call takes up
//            to twice as long: 120001 keys 31 -> 55 us, 15001 9.8 -> 10.9, 200 rows of
//            4200 64 -> 118; where only the first key's scale is such a one, under 1 us.
// A lane's scores are of the row that is its column in both products and of the keys
// that its group of V's layout holds, so nothing moves between lanes but the
// maximum's two exchanges a group.
constexpr float kHeadroom = 4.f, kWeightBits = 10.f;

struct Kv4Attn {
    const float* q;          // [T][ldq], n_heads * D of a row
    const uint8_t *kc, *vc;  // the layer's codes and scales
    const uint16_t *ks, *vs;
    float *out, *part;       // [T][n_heads][D]; [T][n_heads][nch][kv4_part(D)] where nch > 1
    int* ctr;                // a counter a block, zero between launches: the merge in this launch; or null
    size_t codes, scales;    // of a head
    uint16_t* out16;         // the result as bf16 instead of out; or null
    const int* pos_dev;      // T 1: ctx is one more than this (at most ctx); or null
    const float *cos_t, *sin_t;   // [max_seq][D / 2]: q is rotated at its position as it is read; or null
    int n_heads, rep, T, ctx, ldq;
    uint32_t magic;          // floor(2^32 / rep) + 1: row / rep is the high word of row * magic while row * rep < 2^32
    int nch;                 // workgroups that share the keys of a block of rows
    float sl2, qsign;        // |scale| log2(e), the scale's sign
};

__device__ __forceinline__ int kv4_token(const Kv4Attn& a, int row) {
    return a.rep == 1 ? row : (int)__umulhi((uint32_t)row, a.magic);
}

// Row `row` of KV head g among the T * n_heads rows of the result.
__device__ __forceinline__ size_t kv4_row(const Kv4Attn& a, int g, int row) {
    const int t = kv4_token(a, row);
    return (size_t)t * a.n_heads + g * a.rep + (row - t * a.rep);
}

// Four elements of the result from element i on.
__device__ __forceinline__ void kv4_store(float* out, uint16_t* out16, size_t i, const float (&x)[4]) {
    if (out16) {
        const uint2 y = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        __builtin_memcpy(out16 + i, &y, 8);
    } else {
        __builtin_memcpy(out + i, x, 16);
    }
}

__device__ __forceinline__ h2v as_h2(uint32_t u) { return __builtin_bit_cast(h2v, u); }

// 0x6400 twice, in a vector register: v_and_or_b32 takes no literal and one scalar.
__device__ __forceinline__ uint32_t magic1024() {
    uint32_t m = 0x64006400u;
    asm("" : "+v"(m));
    return m;
}

// The eight codes of a word, minus 8, as f16: nibbles (0, 4), (1, 5), (2, 6), (3, 7).
// 0x6400 | n is 1024 + n; with n four bits higher 1024 + 16 n.
__device__ __forceinline__ void codes8(uint32_t w, uint32_t magic, h2v& a, h2v& b, h2v& c, h2v& d) {
    const h2v low = {(_Float16)1032.f, (_Float16)1032.f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f},
              high = {(_Float16)-72.f, (_Float16)-72.f};
    const uint32_t u = w >> 8;
    a = as_h2((w & 0x000F000Fu) | magic) - low;
    b = __builtin_elementwise_fma(as_h2((w & 0x00F000F0u) | magic), sixteenth, high);
    c = as_h2((u & 0x000F000Fu) | magic) - low;
    d = __builtin_elementwise_fma(as_h2((u & 0x00F000F0u) | magic), sixteenth, high);
}

__device__ __forceinline__ h8v h8_of(h2v a, h2v b, h2v c, h2v d) { return h8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; }

// Two f16 pieces of the products x f and y g: together 22 bits.  The first ones pass
// through an empty asm, so that the piece that is subtracted is the one that is
// multiplied: the compiler would form it twice, by a conversion of the rounded
// product and by one that is fused with the product, which now and then differ.
__device__ __forceinline__ void split2(float x, float f, float y, float g, h2v& hi, h2v& lo) {
    float u = fmaf(x, f, 0.f), v = fmaf(y, g, 0.f);
    asm("" : "+v"(u), "+v"(v));
    uint32_t h = __builtin_bit_cast(uint32_t, h2v{(_Float16)u, (_Float16)v});
    asm("" : "+v"(h));
    hi = as_h2(h);
    u = fmaf(x, f, -(float)hi.x), v = fmaf(y, g, -(float)hi.y);
    asm("" : "+v"(u), "+v"(v));
    lo = h2v{(_Float16)u, (_Float16)v};
}

// The same of single values.
__device__ __forceinline__ void split2(float x, float y, h2v& hi, h2v& lo) {
    uint32_t h = __builtin_bit_cast(uint32_t, h2v{(_Float16)x, (_Float16)y});
    asm("" : "+v"(h));
    hi = as_h2(h);
    lo = h2v{(_Float16)(x - (float)hi.x), (_Float16)(y - (float)hi.y)};
}

__device__ __forceinline__ float over_groups_max(float v) {   // over the lanes of a column
    float2 t = swap_rows16(v, v);
    v = fmaxf(t.x, t.y);
    t = swap_halves32(v, v);
    return fmaxf(t.x, t.y);
}

__device__ __forceinline__ float over_groups_sum(float v) {
    float2 t = swap_rows16(v, v);
    v = t.x + t.y;
    t = swap_halves32(v, v);
    return t.x + t.y;
}

// Slots 2j and 2j + 1 of a lane's eight scales.
__device__ __forceinline__ uint32_t word_of(const uint4& x, int j) { return j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w; }

// The 16 NG rows of a wave: q in two pieces, the factor from a score to powers of two,
// running maximum and sum, the number of keys that the lane's rows see, O.
template <int NB, int NG>
struct Kv4Rows {
    h8v qh[NG][NB], ql[NG][NB];
    float factor[NG], m2[NG], l[NG];
    int seen[NG];
    f4v o[NG][2 * NB];
};

// A lane's elements of a row of q (of each block those of its group) and of the tables.
template <int NB>
struct Kv4Query {
    float y[NB][8], cr[NB / 2][8], sr[NB / 2][8];
    int at;   // the row's position
};

template <int NB>
__device__ __forceinline__ void kv4_query(Kv4Query<NB>& x, const Kv4Attn& a, int g, int row, int L) {
    const int t = kv4_token(a, row);
    x.at = a.ctx - a.T + t;
    const float* qp = a.q + (size_t)t * a.ldq + (g * a.rep + (row - t * a.rep)) * (32 * NB) + 8 * L;
#pragma unroll
    for (int b = 0; b < NB; ++b) __builtin_memcpy(x.y[b], qp + 32 * b, 32);
    if (!a.cos_t) return;
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) {
        __builtin_memcpy(x.cr[b], a.cos_t + (size_t)x.at * (16 * NB) + 32 * b + 8 * L, 32);
        __builtin_memcpy(x.sr[b], a.sin_t + (size_t)x.at * (16 * NB) + 32 * b + 8 * L, 32);
    }
}

template <int NB, int NG>
__device__ __forceinline__ void kv4_rows_init(Kv4Rows<NB, NG>& r, const Kv4Attn& a, Kv4Query<NB>& q, int n) {
    float x[NB][8], amax = 0.f;
    if (a.cos_t) {   // a pair's elements are half a head apart: both are the lane's
#pragma unroll
        for (int b = 0; b < NB / 2; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                attn::rope2(q.y[b][e], q.y[b + NB / 2][e], q.cr[b][e], q.sr[b][e], &q.y[b][e], &q.y[b + NB / 2][e]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[b][2 * (e & 3) + (e >> 2)] = q.y[b][e];   // in the order of codes8
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(q.y[b][e]));
    }
    amax = over_groups_max(amax);
    const int k = min(140 - (int)(__float_as_uint(amax) >> 23), 60);
    const float up = a.qsign * __uint_as_float((uint32_t)(k + 127) << 23);
    r.factor[n] = a.sl2 * __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        h2v hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2(x[b][2 * e], up, x[b][2 * e + 1], up, hi[e], lo[e]);
        r.qh[n][b] = h8_of(hi[0], hi[1], hi[2], hi[3]);
        r.ql[n][b] = h8_of(lo[0], lo[1], lo[2], lo[3]);
    }
    r.seen[n] = q.at + 1;
    r.m2[n] = kNegInf;
    r.l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) r.o[n][i] = f4v{};
}

// A row's weights times a block's scales (vs) of 32 keys, formed apart: in two f16 pieces of
// the products times 2^k, the largest of which over the keys lies in [2^14, 2^15); 2^-k is
// returned.  end: as in kv4_weights; a key that the row does not see has no product, so
// that neither its scale nor what it holds matters.  A product that is no number
// stays one (the maximum passes over it).
__device__ __forceinline__ float kv4_apart(const float (&p)[8], const uint4& vs, int end, h2v (&hi)[4], h2v (&lo)[4]) {
    auto product = [&](int e) {   // formed twice: eight held between cost registers that the many-rows kernel has for q
        const h2v d = as_h2(word_of(vs, e >> 1));
        return kv4::key_of(0, e) >= end ? 0.f : p[e] * (float)((e & 1) ? d.y : d.x);
    };
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(product(e)));
    top = over_groups_max(top);
    const int k = min(141 - (int)(__float_as_uint(top) >> 23), 126);
    const float up = __uint_as_float((uint32_t)(127 + k) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // slots (0, 2), (1, 3), (4, 6), (5, 7), as the codes stand
        const int e = 4 * (i >> 1) + (i & 1);
        split2(product(e), up, product(e + 2), up, hi[i], lo[i]);
    }
    return __uint_as_float((uint32_t)(127 - k) << 23);
}

// KG groups of 32 keys from key0 on; src: their operands (k, v) and scales (ks, vs) by
// group and block.  kEdge: some row does not see all of them; kApart: as well, values'
// scales may be of any size (or no number).
enum { kInside, kEdge, kApart };

// A row's scores of KG groups of 32 keys, the lane's, become weights; m2 and l move on, and the
// factor that O so far takes is returned.  end: the first key, from the lane's first one
// on, that the row does not see.
template <int MODE, int KG>
__device__ __forceinline__ float kv4_weights(float (&s)[KG][8], float factor, int end, float& m2, float& l) {
    float mx = kNegInf;
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (MODE != kInside) s[kg][e] = 32 * kg + kv4::key_of(0, e) >= end ? kNegInf : s[kg][e];
            mx = fmaxf(mx, s[kg][e]);
        }
    mx = over_groups_max(mx);
    mx = mx == kNegInf ? kNegInf : mx * factor;
    const bool grow = mx > m2 + kHeadroom;
    const float mn = grow ? mx : m2;
    const float corr = grow ? __builtin_amdgcn_exp2f(m2 - mn) : 1.f;
    m2 = mn;
    const float at = mn == kNegInf ? 0.f : kWeightBits - mn;
    float sum = 0.f;
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[kg][e] = __builtin_amdgcn_exp2f(fmaf(s[kg][e], factor, at));   // 0 of -inf: the factor is positive
            sum += s[kg][e];
        }
    l = fmaf(l, corr, sum);
    return corr;
}

template <int MODE, int KG, int NB, int NG, class Src>
__device__ __forceinline__ void kv4_keys(Kv4Rows<NB, NG>& r, const Src& src, int key0, int L) {
    // ---- scores: slots 4u + j of the lane's keys ----
    // The next half group's operands are read before this one's products (LDS takes longer
    // than a few of those); the barriers hold the order.
    float s[NG][KG][8];
    h8v ka[2][NB];
    h2v dk[2][NB][2];
    auto read = [&](int i) {   // half group i
#pragma unroll
        for (int b = 0; b < NB; ++b) ka[i & 1][b] = src.k(i >> 1, i & 1, b);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint2 ks = src.ks(i >> 1, i & 1, b);
            dk[i & 1][b][0] = as_h2(ks.x);
            dk[i & 1][b][1] = as_h2(ks.y);
        }
    };
    read(0);
#pragma unroll
    for (int i = 0; i < 2 * KG; ++i) {
        if (i + 1 < 2 * KG) read(i + 1);
        if (Src::kValues) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            f4v t[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) t[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[i & 1][b], r.ql[n][b], f4v{}, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < NB; ++b) t[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[i & 1][b], r.qh[n][b], t[b], 0, 0, 0);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float& x = s[n][i >> 1][4 * (i & 1) + j];
                    const h2v d = dk[i & 1][b][j >> 1];
                    x = fmaf(t[b][j], (float)((j & 1) ? d.y : d.x), b == 0 ? 0.f : x);
                }
        }
    }

    if (Src::kValues) __builtin_amdgcn_s_setprio(1);   // the other wave's products run under this one's softmax
    __builtin_amdgcn_sched_barrier(0);   // no loads of the next part early: they would cost registers
    // ---- softmax ----
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        const float corr = kv4_weights<MODE, KG>(s[n], r.factor[n], r.seen[n] - key0 - 4 * L, r.m2[n], r.l[n]);
        // Without a branch around it, although corr is 1 most of the time: the branch keeps
        // O in registers twice.
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) r.o[n][t] *= corr;
    }

    if (Src::kValues) __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    // ---- output ----
    if constexpr (Src::kValues && MODE != kApart) {
        // Whole values stand in two pieces: p alone is split, once for all blocks.
        constexpr int T = 2 * NB, AHEAD = 2;
        h8v ph[KG][NG], pl[KG][NG], vh[AHEAD + 1], vl[AHEAD + 1];
        auto split = [&](int kg, int n) {
            h2v hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = 4 * (i >> 1) + (i & 1);
                split2(s[n][kg][e], s[n][kg][e + 2], hi[i], lo[i]);
            }
            ph[kg][n] = h8_of(hi[0], hi[1], hi[2], hi[3]);
            pl[kg][n] = h8_of(lo[0], lo[1], lo[2], lo[3]);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) src.value(i / T, i % T, vh[i], vl[i]);
#pragma unroll
        for (int n = 0; n < NG; ++n) split(0, n);
#pragma unroll
        for (int i = 0; i < KG * T; ++i) {
            const int kg = i / T, t = i % T, at = i % (AHEAD + 1), next = (i + AHEAD) % (AHEAD + 1);
            if (i + AHEAD < KG * T) src.value((i + AHEAD) / T, (i + AHEAD) % T, vh[next], vl[next]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NG; ++n) r.o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[at], ph[kg][n], r.o[n][t], 0, 0, 0);
#pragma unroll
            for (int n = 0; n < NG; ++n) r.o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[at], pl[kg][n], r.o[n][t], 0, 0, 0);
#pragma unroll
            for (int n = 0; n < NG; ++n) r.o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[at], ph[kg][n], r.o[n][t], 0, 0, 0);
            if (kg + 1 < KG && t < NG) split(kg + 1, t);   // the next group's weights between this one's products
        }
        return;
    }
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            h8v va, wa;   // even elements, odd elements
            src.v(kg, b, va, wa);
            const uint4 vs = src.vs(kg, b);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                h2v hi[4], lo[4];
                float back = 1.f;
                if constexpr (MODE == kApart) {
                    static_assert(KG == 1, "weights of one group of keys");
                    back = kv4_apart(s[n][0], vs, r.seen[n] - key0 - 4 * L, hi, lo) * Src::kUp;
                } else {
                    // Slots (0, 2), (1, 3), (4, 6), (5, 7), as the codes stand.
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * (i >> 1) + (i & 1);
                        const h2v d0 = as_h2(word_of(vs, e >> 1)), d1 = as_h2(word_of(vs, (e >> 1) + 1));
                        split2(s[n][kg][e], (i & 1) ? d0.y : d0.x, s[n][kg][e + 2], (i & 1) ? d1.y : d1.x, hi[i], lo[i]);
                    }
                }
                const h8v ph = h8_of(hi[0], hi[1], hi[2], hi[3]), pl = h8_of(lo[0], lo[1], lo[2], lo[3]);
                if constexpr (MODE == kApart) {
                    f4v t = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, f4v{}, 0, 0, 0);
                    f4v z = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, pl, f4v{}, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph, t, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, ph, z, 0, 0, 0);
                    r.o[n][2 * b] += t * back;
                    r.o[n][2 * b + 1] += z * back;
                } else {
                    r.o[n][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, r.o[n][2 * b], 0, 0, 0);
                    r.o[n][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, pl, r.o[n][2 * b + 1], 0, 0, 0);
                    r.o[n][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph, r.o[n][2 * b], 0, 0, 0);
                    r.o[n][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa, ph, r.o[n][2 * b + 1], 0, 0, 0);
                }
            }
        }
}

// A wave's share of 32 keys as it is loaded: lane (c, L) holds K words of keys c and
// 16 + c, V bytes of elements 2c, 2c + 1 of each block for the keys of group L, and
// those keys' scales, of NS blocks: all, or the one that the lane's column stands for; and one
// word of V's scales of the group L for their size, which the lanes of L look at together.
template <int NB, int NS = NB>
struct Kv4Raw {
    uint32_t kw[2][NB], vw[2 * NB];
    uint4 kd[NS], vd[NS];
    uint32_t two, magic;
    static constexpr bool kValues = false;
    static constexpr float kUp = 1.f;   // what O is held times

    __device__ __forceinline__ void value(int, int, h8v&, h8v&) const {}
    __device__ __forceinline__ h8v k(int, int u, int b) const {
        h2v x0, x1, x2, x3;
        codes8(kw[u][b], magic, x0, x1, x2, x3);
        return h8_of(x0, x1, x2, x3);
    }
    __device__ __forceinline__ void v(int, int b, h8v& even, h8v& odd) const {
        h2v v0, v1, v2, v3, w0, w1, w2, w3;
        codes8(vw[2 * b], magic, v0, w0, v1, w1);        // slots (0, 2), (1, 3)
        codes8(vw[2 * b + 1], magic, v2, w2, v3, w3);    // slots (4, 6), (5, 7)
        even = h8_of(v0, v1, v2, v3);
        odd = h8_of(w0, w1, w2, w3);
    }
    __device__ __forceinline__ uint2 ks(int, int u, int b) const { return u ? make_uint2(kd[b].z, kd[b].w) : make_uint2(kd[b].x, kd[b].y); }
    __device__ __forceinline__ uint4 vs(int, int b) const { return vd[b]; }
};

// Buffer loads from the group's own resources: their addresses cost no vector instructions.
template <int W>
__device__ __forceinline__ void buffer_words(uint32_t (&to)[W], __amdgpu_buffer_rsrc_t r, int at) {
    static_assert(W == 2 || W == 4 || W == 8, "words of a lane");
    if constexpr (W == 2) {
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
        to[0] = x.x;
        to[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at + 4 * i, 0, 0));
            to[i] = x.x;
            to[i + 1] = x.y;
            to[i + 2] = x.z;
            to[i + 3] = x.w;
        }
    }
}

template <class T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t group_buffer(const T* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, bytes, 0x00020000);
}

template <int NB, int NS>
__device__ __forceinline__ void kv4_load(Kv4Raw<NB, NS>& r, const uint8_t* kc, const uint8_t* vc, const uint16_t* ks,
                                         const uint16_t* vs, int kb, int c, int L, int own) {
    constexpr int D = 32 * NB, CODES = kv4::kKeys * D / 2;
    const auto kr = group_buffer(kc + (size_t)kb * CODES, CODES), vr = group_buffer(vc + (size_t)kb * CODES, CODES);
    const auto sr = group_buffer(ks + (size_t)kb * D, 2 * D), tr = group_buffer(vs + (size_t)kb * D, 2 * D);
#pragma unroll
    for (int u = 0; u < 2; ++u) buffer_words<NB>(r.kw[u], kr, (c + 16 * u) * (D / 2) + 4 * L * NB);
#pragma unroll
    for (int b = 0; b < NS; ++b)
        r.kd[b] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(sr, 16 * (L * NB + own + b), 0, 0));
    buffer_words<2 * NB>(r.vw, vr, (L * 16 + c) * 8 * NB);
#pragma unroll
    for (int b = 0; b < NS; ++b)
        r.vd[b] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(tr, 16 * (L * NB + own + b), 0, 0));
    r.two = __builtin_amdgcn_raw_buffer_load_b32(tr, 16 * L * NB + 4 * (c % (4 * NB)), 0, 0);
}

// A chunk's partial of a row: acc[D], m, l and two floats that align the next.  The host
// keeps all of a launch below 2 GiB.
constexpr int kv4_part(int d) { return d + 4; }
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef unsigned int u2v __attribute__((ext_vector_type(2)));

// An offset that is past part_buffer's range for every size of a load: it answers 0.
constexpr int kOutside = (int)0x80000000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_buffer(const float* part) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(part), 0, 0x7fffffff, 0x00020000);
}

// The last workgroup of a block merges its chunks, up to 32 of them (all that its lanes ask
// for at once); more are merged by a launch of their own, a workgroup a row.  In the launch
// / in one of its own, us: 16 chunks (32/4 heads of 64, 4096 keys) 6.3 / 8.0, 6 (32/8 of 128, 1500) 6.8
// / 8.1, 32 (15001) 10.0 / 11.3, 32 (120001) 34.2 / 36.3, 3 (40 rows of 3001) 16.4 / 18.0; a merge in
// the launch of any number took, 59 chunks (8/1 of 128, 15001), 12.9 / 10.3, 235 (60001) 26.5 / 11.9.
constexpr int kMergedChunks = 32;

// ---- few rows ---------------------------------------------------------------------
// In a block of 16 / NB rows (a decode step of a usual group) the 16 columns stand for
// its rows and a head's blocks: column NB row + b has the row's q where its block
// is b, zeros elsewhere, and the weights times b's scales of V.  So a lane loads, splits and
// scales one block of q and of the scales instead of all, which is most of the work of a
// group of keys; the columns' scores of a row are summed by exchanges within four lanes,
// and of each block's product O the column with the block's own scales is kept.  One
// row of 1500, 15001 and 120001 keys at 32/8 heads of 128: 7.9, 11.4 and 40 us with a column
// a row, 6.8, 10.0 and 34.5 so; 4096 keys at 32/4 of 64 6.6 and 6.3.
template <int NB>
struct Kv4Few {
    h8v qh[NB], ql[NB];
    float factor, m2, l;
    int seen;
    f4v o[2 * NB];
};

template <int NB>
__device__ __forceinline__ float over_blocks_max(float v) {
    v = fmaxf(v, quad_f(v, 1));
    return NB == 4 ? fmaxf(v, quad_f(v, 2)) : v;
}

template <int NB>
__device__ __forceinline__ float over_blocks_sum(float v) {
    v += quad_f(v, 1);
    return NB == 4 ? v + quad_f(v, 2) : v;
}

// b: the lane's block.
template <int NB>
__device__ __forceinline__ void kv4_few_init(Kv4Few<NB>& r, const Kv4Attn& a, int g, int row, int b, int L) {
    const int t = kv4_token(a, row), at = a.ctx - a.T + t;
    const float* qp = a.q + (size_t)t * a.ldq + (g * a.rep + (row - t * a.rep)) * (32 * NB) + 8 * L;
    float y[8], amax = 0.f;
    __builtin_memcpy(y, qp + 32 * b, 32);
    if (a.cos_t) {
        const bool first = b < NB / 2;   // of a pair, whose elements are half a head apart
        const int i = first ? b : b - NB / 2;
        float x[8], cr[8], sr[8];
        __builtin_memcpy(x, qp + 32 * (first ? b + NB / 2 : i), 32);
        __builtin_memcpy(cr, a.cos_t + (size_t)at * (16 * NB) + 32 * i + 8 * L, 32);
        __builtin_memcpy(sr, a.sin_t + (size_t)at * (16 * NB) + 32 * i + 8 * L, 32);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float u, v;
            attn::rope2(first ? y[e] : x[e], first ? x[e] : y[e], cr[e], sr[e], &u, &v);
            y[e] = first ? u : v;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(y[e]));
    amax = over_blocks_max<NB>(over_groups_max(amax));
    const int k = min(140 - (int)(__float_as_uint(amax) >> 23), 60);
    const float up = a.qsign * __uint_as_float((uint32_t)(k + 127) << 23);
    r.factor = a.sl2 * __uint_as_float((uint32_t)(127 - k) << 23);
    h2v hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split2(y[e], up, y[e + 4], up, hi[e], lo[e]);   // in the order of codes8
    const h8v qh = h8_of(hi[0], hi[1], hi[2], hi[3]), ql = h8_of(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        r.qh[i] = i == b ? qh : h8v{};
        r.ql[i] = i == b ? ql : h8v{};
    }
    r.seen = at + 1;
    r.m2 = kNegInf;
    r.l = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) r.o[i] = f4v{};
}

template <int MODE, int NB>
__device__ __forceinline__ void kv4_few_keys(Kv4Few<NB>& r, const Kv4Raw<NB, 1>& x, int key0, int L) {
    f4v t[2] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const h8v k = x.k(0, u, b);
            t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, r.ql[b], t[u], 0, 0, 0);
            t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, r.qh[b], t[u], 0, 0, 0);
        }
    float s[1][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const h2v d = as_h2(word_of(x.kd[0], e >> 1));
        s[0][e] = over_blocks_sum<NB>(t[e >> 2][e & 3] * (float)((e & 1) ? d.y : d.x));
    }
    const float corr = kv4_weights<MODE, 1>(s, r.factor, r.seen - key0 - 4 * L, r.m2, r.l);
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) r.o[i] *= corr;
    h2v hi[4], lo[4];
    float back = 1.f;   // of the column's products, formed apart
    if constexpr (MODE == kApart) {
        back = kv4_apart(s[0], x.vd[0], r.seen - key0 - 4 * L, hi, lo);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // slots (0, 2), (1, 3), (4, 6), (5, 7), as the codes stand
            const int e = 4 * (i >> 1) + (i & 1);
            const h2v d0 = as_h2(word_of(x.vd[0], e >> 1)), d1 = as_h2(word_of(x.vd[0], (e >> 1) + 1));
            split2(s[0][e], (i & 1) ? d0.y : d0.x, s[0][e + 2], (i & 1) ? d1.y : d1.x, hi[i], lo[i]);
        }
    }
    const h8v ph = h8_of(hi[0], hi[1], hi[2], hi[3]), pl = h8_of(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        h8v v[2];   // even elements, odd elements
        x.v(0, b, v[0], v[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f4v& o = r.o[2 * b + h];
            if constexpr (MODE == kApart) {
                f4v y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], pl, f4v{}, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], ph, y, 0, 0, 0);
                o += y * back;
            } else {
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], pl, o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], ph, o, 0, 0, 0);
            }
        }
    }
}

constexpr int kWaves = 8;   // of a workgroup that has a CU to itself; half of them where two share it

template <int D, int ROWS, int W>
struct Kv4WavesLds {
    float o[W][ROWS * (D + 4)], m[ROWS][W], l[ROWS][W];
};

template <int D, bool FEW, int W>
__global__ __launch_bounds__(64 * W, 2) void kv4_attn_rows_kernel(Kv4Attn a) {
    constexpr int NB = D / 32, ROWS = FEW ? 16 / NB : 16, OS = D + 4;
    __shared__ int last;
    __shared__ __align__(16) Kv4WavesLds<D, ROWS, W> x;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, L = lane >> 4;
    const int lane_row = FEW ? c / NB : c, own = FEW ? c % NB : 0;   // the lane's row, its block
    if (a.pos_dev) a.ctx = min(*a.pos_dev + 1, a.ctx);
    const int nch = a.nch, chunk = blockIdx.x, g = blockIdx.y, row0 = blockIdx.z * ROWS, R = a.T * a.rep;
    const uint8_t *kc = a.kc + g * a.codes, *vc = a.vc + g * a.codes;
    const uint16_t *ks = a.ks + g * a.scales, *vs = a.vs + g * a.scales;
    // Keys that the block's first and last row see.
    const int past = a.ctx - a.T + 1, fewest = past + kv4_token(a, row0), most = past + kv4_token(a, min(row0 + ROWS - 1, R - 1));
    // The wave's groups of keys: every nch * W-th, so that all share any context alike.
    const int kb0 = chunk * W + w, stride = nch * W;
    auto mine_of = [&](int groups) { return groups > kb0 ? (groups - kb0 + stride - 1) / stride : 0; };
    const int mine = mine_of((most + kv4::kKeys - 1) / kv4::kKeys), inside = min(mine, mine_of(fewest / kv4::kKeys));

    using Raw = Kv4Raw<NB, FEW ? 1 : NB>;
    Raw raw;
    raw.magic = magic1024();
    if (mine > 0) kv4_load(raw, kc, vc, ks, vs, kb0, c, L, own);
    __builtin_amdgcn_sched_barrier(0);
    std::conditional_t<FEW, Kv4Few<NB>, Kv4Rows<NB, 1>> r;
    const int row = min(row0 + lane_row, R - 1);   // rows past the last one repeat it and are not stored
    if constexpr (FEW) {
        kv4_few_init(r, a, g, row, own, L);
    } else {
        Kv4Query<NB> q;
        kv4_query(q, a, g, row, L);
        kv4_rows_init(r, a, q, 0);
    }
    auto keys = [&](auto mode, const Raw& x, int i) {
        const int key0 = (kb0 + i * stride) * kv4::kKeys;
        if constexpr (FEW) kv4_few_keys<mode.value>(r, x, key0, L);
        else kv4_keys<mode.value, 1>(r, x, key0, L);
    };
    constexpr std::integral_constant<int, kInside> whole;
    constexpr std::integral_constant<int, kEdge> edge;
    constexpr std::integral_constant<int, kApart> apart;
    // Three loops of one body each (two in one would cost each other registers): the groups
    // that every row sees whole, those at some row's edge, and those of both that the first
    // two left because of a scale, which the third looks for between the first and the last of them.
    int from = mine, to = 0;
    // Of the lane's two scales one is 2 or more or no number (exponent bits 1xxxx), or below
    // 2^-11 (000xx) and not 0.
    auto is_apart = [&](const Raw& x) {
        const uint32_t m = x.two & 0x7FFF7FFFu, not0 = (m + 0x7FFF7FFFu) >> 2;
        return __builtin_amdgcn_ballot_w64(((m & 0x40004000u) | (not0 & ~(m | m << 1) & 0x20002000u)) != 0) != 0;
    };
    auto load = [&](int i) { kv4_load(raw, kc, vc, ks, vs, kb0 + i * stride, c, L, own); };   // i < mine
    int i = 0;
    for (; i < inside; ++i) {
        const Raw cur = raw;
        if (i + 1 < mine) load(i + 1);
        if (is_apart(cur)) from = min(from, i), to = i + 1;
        else keys(whole, cur, i);
    }
    for (; i < mine; ++i) {
        const Raw cur = raw;
        if (i + 1 < mine) load(i + 1);
        if (is_apart(cur)) from = min(from, i), to = i + 1;
        else keys(edge, cur, i);
    }
    if (from < to) load(from);
    for (i = from; i < to; ++i) {
        const Raw cur = raw;
        if (i + 1 < to) load(i + 1);
        if (is_apart(cur)) keys(apart, cur, i);
    }

    // ---- the waves' results, then the chunk's ----
    float l, m;
    if constexpr (FEW) l = r.l, m = r.m2;
    else l = r.l[0], m = r.m2[0];
    l = over_groups_sum(l);
    if (L == 0 && own == 0) {
        x.m[lane_row][w] = l != l ? INFINITY : m;   // a NaN has to win where the others' weights would drop it
        x.l[lane_row][w] = l;
    }
    // Rows 4L + j of a block's two tiles: its elements 8L + 2j and 8L + 2j + 1.
    auto put = [&](int b, const f4v& even, const f4v& odd) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float4*>(&x.o[w][lane_row * OS + 32 * b + 8 * L + 4 * h]) =
                make_float4(even[2 * h], odd[2 * h], even[2 * h + 1], odd[2 * h + 1]);
    };
    if constexpr (FEW) {
        f4v even = r.o[0], odd = r.o[1];
#pragma unroll
        for (int b = 1; b < NB; ++b) {
            even = own == b ? r.o[2 * b] : even;
            odd = own == b ? r.o[2 * b + 1] : odd;
        }
        put(own, even, odd);
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) put(b, r.o[0][2 * b], r.o[0][2 * b + 1]);
    }
    __syncthreads();
    const int rows = min(ROWS, R - row0), tid = threadIdx.x;
    for (int i = tid; i < rows * (D / 4); i += 64 * W) {
        const int j = i / (D / 4), e = 4 * (i % (D / 4));
        float m[W], M = kNegInf, l = 0.f, v[4] = {};
#pragma unroll
        for (int k = 0; k < W; ++k) M = fmaxf(M, m[k] = x.m[j][k]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = m[k] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[k] - M);
            const float4 y = *reinterpret_cast<const float4*>(&x.o[k][j * OS + e]);
            l = fmaf(f, x.l[j][k], l);
            v[0] = fmaf(f, y.x, v[0]); v[1] = fmaf(f, y.y, v[1]); v[2] = fmaf(f, y.z, v[2]); v[3] = fmaf(f, y.w, v[3]);
        }
        const size_t at = kv4_row(a, g, row0 + j);
        if (nch == 1) {
            const float by = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] *= by;
            kv4_store(a.out, a.out16, at * D + e, v);
            continue;
        }
        // Past this die's L2 (sc1): read by another workgroup of this launch.
        const int p = (int)(4 * ((at * nch + chunk) * kv4_part(D) + e));
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4v, make_float4(v[0], v[1], v[2], v[3])), part_buffer(a.part), p, 0, 16);
        if (e == 0)
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2v, make_float2(M, l)), part_buffer(a.part), p + 4 * D, 0, 16);
    }
    if (nch == 1 || !a.ctr) return;

    // ---- the workgroup that comes last merges the block's chunks, in their order ----
    __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's stores acknowledged (vmcnt 0)
    __syncthreads();
    if (tid == 0) {
        int* ctr = a.ctr + (size_t)(blockIdx.z * gridDim.y + g) * kSmallTileCtrStride;
        last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nch - 1;
        if (last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    // A wave a row, in few instructions: they run once, from a cold cache.  Lane i weighs chunk
    // i; the wave's halves (quarters where D is 64) take every second (fourth) chunk's O,
    // all loads at once.  What lies past the last chunk reads as 0, out of the buffer's range.
    constexpr int Q = D / 4, SHARES = 64 / Q, EACH = kMergedChunks / SHARES, PS = kv4_part(D);
    const auto pr = part_buffer(a.part);
    const int e = 4 * (lane % Q), share = lane / Q;
    for (int j = w; j < rows; j += W) {
        const size_t at = kv4_row(a, g, row0 + j);
        const int first = (int)(4 * at * nch * PS);
        const float2 ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(pr, lane < nch ? first + 4 * (lane * PS + D) : kOutside, 0, 16));
        f4v y[EACH], o = {};
        auto ask = [&](int from) {
#pragma unroll
            for (int i = from; i < from + EACH / 2; ++i) {
                const int k = share + i * SHARES;
                y[i] = __builtin_bit_cast(f4v, __builtin_amdgcn_raw_buffer_load_b128(pr, k < nch ? first + 4 * (k * PS + e) : kOutside, 0, 16));
            }
        };
        ask(0);
        const bool more = nch > EACH / 2 * SHARES;
        if (more) ask(EACH / 2);
        const float m = lane < nch ? ml.x : kNegInf, M = wave_max(m);
        const float f = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - M), l = wave_sum(f * ml.y);
        auto add = [&](int from) {
#pragma unroll
            for (int i = from; i < from + EACH / 2; ++i) o += __shfl(f, share + i * SHARES) * y[i];
        };
        add(0);
        if (more) add(EACH / 2);
        const float by = l == 0.f ? 0.f : 1.f / l;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 t = swap_halves32(o[i], o[i]);
            v[i] = t.x + t.y;
            if (SHARES == 4) {
                t = swap_rows16(v[i], v[i]);
                v[i] = t.x + t.y;
            }
            v[i] *= by;
        }
        if (share == 0) kv4_store(a.out, a.out16, at * D + e, v);
    }
}

// ---- many rows --------------------------------------------------------------------
// Four waves of 32 rows share what they read: a stage of 8192 / D keys is decoded once,
// into LDS, where the operands stand as the lanes read them (a wave decodes a quarter of
// the stage's K and of its V).  The next stage's codes are in registers meanwhile; the
// other workgroup of the CU computes while this one decodes.  Values stand whole, as two
// f16 pieces whose sum is exactly the code times the scale (15 bits) times 2^8, while the
// scale is below 32, so that only p is split, once for all blocks: three products for two, but
// a quarter of the conversions, which cost more (16 cycles a weight and block).  The 2^8,
// which O carries and the last division takes back, lifts values of small scales out of
// f16's subnormal range, whose products lose bits in the matrix cores' sums (values of
// 1e-6: results 1e-5 off without it, as others with it).  Stages with a larger scale, or
// one that is no number, come last, with codes and scales apart.
// Each wave keeps its rows to the end, so nothing is merged.  Three passes, as above.
// 1777 rows of 4001 keys at 32/8 heads of 128 225 us: 0.40 PFLOP/s of the attention's own
// 91 GFLOP, 1.0 of the f16 products (two for a score, three for an output) where a
// large product alone reaches 1.17.  Counted over all SIMDs and the whole launch, matrix
// instructions take 36 % and other vector ones 35 %, the CUs hold work 76 % of the time:
// the two hardly overlap.  At d_head 64 (2500 rows of 2500 at 32/4 heads 97 us) 24 and 34 %
// of 64 %: half the products a key, but the same softmax and split of p.  A third product for
// the scores in place of the scaling (K whole, in two pieces) took as long, one product for
// each took 28 % less.
constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves;
constexpr float kTileUp = 256.f;

template <int NB>
struct Kv4Stage {
    static constexpr int GROUPS = 8 / NB, KEYS = 32 * GROUPS;
    uint4 k[16][64];               // [group][2][NB][lane]
    uint4 v[2][16][64];            // pieces of [group][NB][2][lane]; apart: codes in the first
    uint4 kd[32], vd[32];          // [group][L][block]; vd: apart only
    uint32_t large[kTileWaves];    // a scale of 32 or more among the wave's values
};

template <int NB>
struct Kv4FromStage {
    const Kv4Stage<NB>& st;
    int group, lane;
    static constexpr bool kValues = true;
    static constexpr float kUp = kTileUp;
    __device__ __forceinline__ h8v k(int kg, int u, int b) const {
        return __builtin_bit_cast(h8v, st.k[(2 * (group + kg) + u) * NB + b][lane]);
    }
    __device__ __forceinline__ void value(int kg, int t, h8v& hi, h8v& lo) const {
        hi = __builtin_bit_cast(h8v, st.v[0][2 * (group + kg) * NB + t][lane]);
        lo = __builtin_bit_cast(h8v, st.v[1][2 * (group + kg) * NB + t][lane]);
    }
    __device__ __forceinline__ void v(int kg, int b, h8v& even, h8v& odd) const {
        even = __builtin_bit_cast(h8v, st.v[0][2 * ((group + kg) * NB + b)][lane]);
        odd = __builtin_bit_cast(h8v, st.v[0][2 * ((group + kg) * NB + b) + 1][lane]);
    }
    __device__ __forceinline__ uint2 ks(int kg, int u, int b) const {
        return reinterpret_cast<const uint2*>(&st.kd[(4 * (group + kg) + (lane >> 4)) * NB + b])[u];
    }
    __device__ __forceinline__ uint4 vs(int kg, int b) const { return st.vd[(4 * (group + kg) + (lane >> 4)) * NB + b]; }
};

template <int D>
__global__ __launch_bounds__(64 * kTileWaves, 2) void kv4_attn_tiles_kernel(Kv4Attn a) {
    constexpr int NB = D / 32, NG = 2, ROWS = 16 * NG;
    using Stage = Kv4Stage<NB>;
    constexpr int PAIRS = Stage::GROUPS / 2;
    __shared__ Stage st;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, L = lane >> 4;
    const int g = blockIdx.x, R = a.T * a.rep, past = a.ctx - a.T + 1;
    // The first workgroups, one a CU, take the longest rows from the last block down; the
    // others the shortest ones up.
    const int nblk = gridDim.y, ahead = min(nblk, (256 + (int)gridDim.x - 1) / (int)gridDim.x), y = blockIdx.y;
    const int block = y < ahead ? nblk - 1 - y : y - ahead;
    const int row0 = block * kTileRows + ROWS * w;
    auto keys_of = [&](int row) { return past + kv4_token(a, min(row, R - 1)); };
    const int most = row0 < R ? keys_of(row0 + ROWS - 1) : 0;
    const int end = (keys_of(block * kTileRows + kTileRows - 1) + Stage::KEYS - 1) / Stage::KEYS;
    const int inside = keys_of(block * kTileRows) / Stage::KEYS;   // stages below it are whole for every row

    // This wave's runs of a stage: 1 KiB of K and of V (two blocks of a group of keys), the
    // scales of those values, and (lanes 0..7) a quarter of K's.
    const uint8_t *kc = a.kc + g * a.codes, *vc = a.vc + g * a.codes;
    const uint16_t *ks = a.ks + g * a.scales, *vs = a.vs + g * a.scales;
    const uint32_t magic = magic1024();
    const int vgroup = D == 64 ? w : w >> 1, vblock = D == 64 ? 0 : 2 * (w & 1);
    uint32_t kw[4], vw[4];
    uint4 kd, vd[2];
    auto fetch = [&](int s) {   // past the cache's end: zeros
        const size_t at = (size_t)s * 4096, sat = (size_t)s * 256;   // bytes of codes, f16 scales
        const int left = (int)min((size_t)4096, a.codes - at), sleft = (int)min((size_t)256, a.scales - sat) * 2;
        const auto kr = group_buffer(kc + at, left), vr = group_buffer(vc + at, left);
        const auto sr = group_buffer(ks + sat, sleft), tr = group_buffer(vs + sat, sleft);
        if constexpr (D == 64) {   // a run of K holds both halves of a group's keys, 8 bytes a lane
            uint32_t x[2], y[2];
            buffer_words<2>(x, kr, 1024 * w + c * 32 + 8 * L);
            buffer_words<2>(y, kr, 1024 * w + (c + 16) * 32 + 8 * L);
            kw[0] = x[0]; kw[1] = x[1]; kw[2] = y[0]; kw[3] = y[1];
        } else {
            buffer_words<4>(kw, kr, 1024 * w + c * 64 + 16 * L);
        }
        buffer_words<4>(vw, vr, 32 * (D / 2) * vgroup + (L * 16 + c) * 8 * NB + 8 * vblock);
        kd = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(sr, 16 * (8 * w + (lane & 7)), 0, 0));
#pragma unroll
        for (int j = 0; j < 2; ++j)
            vd[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(tr, 16 * ((4 * vgroup + L) * NB + vblock + j), 0, 0));
    };
    auto put = [&](auto apart) {
        h2v x0, x1, x2, x3, y0, y1, y2, y3;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            codes8(kw[j], magic, x0, x1, x2, x3);
            st.k[4 * w + j][lane] = __builtin_bit_cast(uint4, h8_of(x0, x1, x2, x3));
        }
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            codes8(vw[2 * j], magic, x0, x1, x2, x3);
            codes8(vw[2 * j + 1], magic, y0, y1, y2, y3);
            const int t = 4 * w + 2 * j;   // even elements; odd ones in t + 1
            if constexpr (decltype(apart)::value) {
                st.v[0][t][lane] = __builtin_bit_cast(uint4, h8_of(x0, x2, y0, y2));
                st.v[0][t + 1][lane] = __builtin_bit_cast(uint4, h8_of(x1, x3, y1, y3));
                if (c == 0) st.vd[(4 * vgroup + L) * NB + vblock + j] = vd[j];
            } else {
                // The scales of slots (0, 2), (1, 3), (4, 6), (5, 7), as the codes stand.
                const h2v up = {(_Float16)kTileUp, (_Float16)kTileUp};
                const h2v d0 = as_h2(__builtin_amdgcn_perm(vd[j].y, vd[j].x, 0x05040100)) * up, d1 = as_h2(__builtin_amdgcn_perm(vd[j].y, vd[j].x, 0x07060302)) * up;
                const h2v d2 = as_h2(__builtin_amdgcn_perm(vd[j].w, vd[j].z, 0x05040100)) * up, d3 = as_h2(__builtin_amdgcn_perm(vd[j].w, vd[j].z, 0x07060302)) * up;
                auto both = [&](int to, h2v a0, h2v a1, h2v a2, h2v a3) {
                    const h2v h0 = a0 * d0, h1 = a1 * d1, h2 = a2 * d2, h3 = a3 * d3;
                    st.v[0][to][lane] = __builtin_bit_cast(uint4, h8_of(h0, h1, h2, h3));
                    st.v[1][to][lane] = __builtin_bit_cast(uint4, h8_of(__builtin_elementwise_fma(a0, d0, -h0), __builtin_elementwise_fma(a1, d1, -h1),
                                                                        __builtin_elementwise_fma(a2, d2, -h2), __builtin_elementwise_fma(a3, d3, -h3)));
                };
                both(t, x0, x2, y0, y2);
                both(t + 1, x1, x3, y1, y3);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // exponent bits 1x1xx or 11xxx: 32 and more
                const uint32_t x = word_of(vd[j], i);
                big |= x & (x << 1 | x << 2);
            }
        }
        if (lane < 8) st.kd[8 * w + lane] = kd;
        const bool any = __builtin_amdgcn_ballot_w64((big & 0x40004000u) != 0) != 0;
        if (lane == 0) st.large[w] = any;
    };
    // The stages [from, to): body(s) with each one in LDS.
    auto stages = [&](auto apart, int from, int to, auto body) {
        if (from >= to) return;
        fetch(from);
        for (int s = from; s < to; ++s) {
            __syncthreads();   // every wave has read the stage before
            put(apart);
            if (s + 1 < to) fetch(s + 1);
            __syncthreads();
            body(s);
        }
    };
    auto is_large = [&]() { return __builtin_amdgcn_readfirstlane(st.large[0] | st.large[1] | st.large[2] | st.large[3]) != 0; };

    Kv4Rows<NB, NG> r;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        Kv4Query<NB> q;
        kv4_query<NB>(q, a, g, min(row0 + 16 * n + c, R - 1), L);   // rows past the last one repeat it and are not stored
        kv4_rows_init<NB, NG>(r, a, q, n);
    }
    int from = end, to = 0;   // the stages left for the last pass lie between
    stages(std::false_type(), 0, inside, [&](int s) {
        if (is_large()) {
            from = min(from, s), to = s + 1;
            return;
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
            kv4_keys<kInside, 2>(r, Kv4FromStage<NB>{st, 2 * i, lane}, s * Stage::KEYS + 64 * i, L);
    });
    stages(std::false_type(), inside, end, [&](int s) {
        if (is_large()) {
            from = min(from, s), to = s + 1;
            return;
        }
#pragma unroll 1
        for (int i = 0; i < PAIRS; ++i) {
            const int key0 = s * Stage::KEYS + 64 * i;
            if (key0 < most) kv4_keys<kEdge, 2>(r, Kv4FromStage<NB>{st, 2 * i, lane}, key0, L);
        }
    });
    stages(std::true_type(), from, to, [&](int s) {
        if (!is_large()) return;
#pragma unroll 1
        for (int i = 0; i < Stage::GROUPS; ++i) {
            const int key0 = s * Stage::KEYS + 32 * i;
            if (key0 < most) kv4_keys<kApart, 1>(r, Kv4FromStage<NB>{st, i, lane}, key0, L);
        }
    });
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        const float sum = over_groups_sum(r.l[n]);
        const int row = row0 + 16 * n + c;
        if (row >= R) continue;
        const size_t at = kv4_row(a, g, row);
        const float by = sum == 0.f ? 0.f : 1.f / (sum * kTileUp);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float x[4] = {r.o[n][2 * b][2 * h] * by, r.o[n][2 * b + 1][2 * h] * by, r.o[n][2 * b][2 * h + 1] * by,
                                    r.o[n][2 * b + 1][2 * h + 1] * by};
                kv4_store(a.out, a.out16, at * D + 32 * b + 8 * L + 4 * h, x);
            }
    }
}

// The merge as a launch of its own: a row a workgroup.
// out[row] = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M) l_c over the nch chunks of a row.  A
// thread takes four elements of every P-th chunk, eight at a time whose loads are all issued
// before any is used; they merge through LDS.
template <int D>
__global__ __launch_bounds__(512) void kv4_merge_kernel(const float* __restrict__ part, int nch, float* __restrict__ out,
                                                        uint16_t* __restrict__ out16) {
    constexpr int B = 8, Q = D / 4, P = 512 / Q, PS = kv4_part(D);
    __shared__ float4 so[512];
    __shared__ float sm[P], sl[P];
    const int tid = threadIdx.x, share = tid / Q, i = tid % Q;
    const float* row = part + (size_t)blockIdx.x * nch * PS;
    float M = kNegInf, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = share; c0 < nch; c0 += B * P) {
        float pm[B], pl[B], mb = M;
        float4 po[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const float* x = row + min(c0 + b * P, nch - 1) * PS;
            pm[b] = x[D];
            pl[b] = x[D + 1];
            po[b] = *reinterpret_cast<const float4*>(x + 4 * i);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) mb = fmaxf(mb, pm[b]);   // a repeated last chunk does no harm
        const float f = M == kNegInf ? 0.f : __builtin_amdgcn_exp2f(M - mb);
        sum *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const float e = c0 + b * P < nch && pm[b] != kNegInf ? __builtin_amdgcn_exp2f(pm[b] - mb) : 0.f;
            sum = fmaf(e, pl[b], sum);
            o.x = fmaf(e, po[b].x, o.x); o.y = fmaf(e, po[b].y, o.y); o.z = fmaf(e, po[b].z, o.z); o.w = fmaf(e, po[b].w, o.w);
        }
        M = mb;
    }
    so[tid] = o;
    if (i == 0) {
        sm[share] = M;
        sl[share] = sum;
    }
    __syncthreads();
    if (share) return;
    for (int k = 0; k < P; ++k) M = fmaxf(M, sm[k]);
    float l = 0.f, v[4] = {};
    for (int k = 0; k < P; ++k) {
        const float f = sm[k] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(sm[k] - M);
        const float4 x = so[k * Q + i];
        l = fmaf(f, sl[k], l);
        v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= by;
    kv4_store(out, out16, (size_t)blockIdx.x * D + 4 * i, v);
}

}  // namespace

// Blocks of a row that a workgroup takes: all of them at d_head 64 and 128.
#define VH_KV4_BLOCKS(nb, LAUNCH) \
    if ((nb) % 4 == 0) {          \
        LAUNCH(4);                \
    } else if ((nb) % 2 == 0) {   \
        LAUNCH(2);                \
    } else {                      \
        LAUNCH(1);                \
    }

int launch_kv4_append(hipStream_t s, const KVLayer& L, int n_kv, int d_head, int max_seq, const float* k, const float* v,
                      int T, int pos, const Kv4Model* m) {
    VH_ARG(T >= 1 && n_kv >= 1 && n_kv <= 65535 && d_head >= 32 && d_head % 32 == 0, "kv_append: bad shape");
    VH_ARG(pos >= 0 && T <= max_seq - pos, "kv_append: %d rows at %d beyond max_seq %d", T, pos, max_seq);
    VH_ARG(!m || (m->cos_t && m->sin_t && m->ld >= n_kv * d_head && (!m->pos_dev || T == 1)), "kv_append: bad model call");
    Kv4Append a;
    a.k = k;
    a.v = v;
    a.kc = reinterpret_cast<uint8_t*>(L.k);
    a.vc = reinterpret_cast<uint8_t*>(L.v);
    a.ks = reinterpret_cast<uint16_t*>(L.ks);
    a.vs = reinterpret_cast<uint16_t*>(L.vs);
    a.ld = m ? m->ld : n_kv * d_head;
    a.pos_dev = m ? m->pos_dev : nullptr;
    a.cos_t = m ? m->cos_t : nullptr;
    a.sin_t = m ? m->sin_t : nullptr;
    a.D = d_head;
    a.n_kv = n_kv;
    a.max_seq = max_seq;
    a.T = T;
    a.pos = pos;
    const int groups = (pos + T - 1) / kv4::kKeys - pos / kv4::kKeys + 1, nb = d_head / 32;
    VH_ARG((size_t)groups * n_kv < (1u << 23), "kv_append: %d rows of %d heads are beyond a launch", T, n_kv);
#define VH_APPEND(CB, R) VH_LAUNCH((kv4_append_kernel<CB, R>), dim3(groups * n_kv, 1, 2 * (nb / CB)), dim3(128 * CB), 0, s, a)
#define VH_APPEND_AS(CB) VH_APPEND(CB, false)
    if (m) {   // d_head 64 or 128
        if (nb == 4) VH_APPEND(4, true);
        else VH_APPEND(2, true);
    } else {
        VH_KV4_BLOCKS(nb, VH_APPEND_AS)
    }
#undef VH_APPEND_AS
#undef VH_APPEND
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

int launch_kv4_dequant(hipStream_t s, const KVLayer& L, int n_kv, int d_head, int max_seq, int ctx_len, float* K,
                       float* V) {
    VH_ARG(ctx_len >= 1 && ctx_len <= max_seq, "kv_dequant: ctx_len %d outside [0,%d]", ctx_len, max_seq);
    const int groups = (ctx_len + kv4::kKeys - 1) / kv4::kKeys, nb = d_head / 32;
    VH_ARG((size_t)groups * n_kv < (1u << 23), "kv_dequant: %d rows of %d heads are beyond a launch", ctx_len, n_kv);
#define VH_DEQUANT(CB)                                                                                              \
    VH_LAUNCH(kv4_dequant_kernel<CB>, dim3(groups * n_kv, 1, nb / CB), dim3(256), 0, s, reinterpret_cast<const uint8_t*>(L.k), \
              reinterpret_cast<const uint8_t*>(L.v), reinterpret_cast<const uint16_t*>(L.ks),                       \
              reinterpret_cast<const uint16_t*>(L.vs), n_kv * d_head, d_head, max_seq, ctx_len, K, V)
    VH_KV4_BLOCKS(nb, VH_DEQUANT)
#undef VH_DEQUANT
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

namespace {
struct Kv4Plan {
    bool tiles = false;                      // the kernel for many rows
    bool few = false;                        // the kernel for a column a row and block
    int waves = kWaves;                      // of a block of 16 rows
    int blocks = 1, nch = 1;                 // blocks of rows of a KV head, workgroups that share a block's keys
};

// Tiles or blocks of 16 rows: whichever is estimated to take less.  A block of 16 rows costs a
// fixed time and each of its rows' keys another; tiles that stand alone on a CU take a time a key of the
// longest row, where some share one a little more, and where there are many the CUs are evenly
// full.  In us, fitted to 362 pairs of times (T 200 to 6400, contexts from T to T + 6000, 11 layouts): the
// choice costs 0.1 % on average and 10 % at most, where a limit on the number of tiles cost 1 to
// 3 % and 43 % (a prompt of 3700 tokens at 8/8 heads of 128: 119 in blocks, 176 in 232 tiles, of which
// the longest take all the time; 900 of 4900 at 32/8, as many: 248 and 233).
// In blocks, the keys are shared out to as many workgroups as there are CUs, one group of keys
// or more for each wave.  With 128, 256, 384 and 512 workgroups in all, us: one row at 32/8 heads of 128
// of 15001 keys 11.8, 10.0, 14.4, 13.5, of 120001 51, 34, 42, 39; 40 rows of 3001 keys 27, 16, 26, 23
// (one stands on a CU at a time).
// Blocks of few rows, whose groups of keys cost less but are read once more for each, where
// that is one block or all of them stand on the CUs at once with up to four groups a wave.  With 16
// rows / few, us, at 32/8 heads of 128: 5 rows of 3000 keys (2 groups) 10.1 / 8.4, of 6000 (4)
// 12.3 / 11.6, 8 of 3000 (3) 10.9 / 10.1, of 6000 (6) 12.4 / 14.7, 21 of 700 (3) 9.8 / 8.2, of 1500
// (6) 11.6 / 12.6, 48 of 250 (384 blocks) 7.0 / 8.5; at 32/4 of 64: 64 of 700 (3) 8.7 / 6.7,
// 233 of 700 (932 blocks) 10.4 / 14.4.
// Where there are more blocks of 16 rows than CUs each has four waves instead of eight, and one
// block's start and end run beside another's keys; at d_head 64 two of eight stand on a CU anyway, so
// that only short contexts gain.  With 8 / 4 waves, us, at 32/8 heads of 128: 200 rows of 500 keys (400
// blocks) 15.6 / 12.2, of 4200 66.5 / 63.6, 400 of 700 32.6 / 24.1, 100 of 1100 (200 blocks) 13.2 / 13.8; at
// 32/4 of 64: 400 rows of 400 11.3 / 8.7, of 1400 24.7 / 23.8, of 4400 67.9 / 68.9.
constexpr long kSharers = 256, kFewGroups = 4, kFourFrom64 = 2048;

struct Kv4Cost {
    double block, pairs;             // a workgroup of 16 rows, a million keys of a row
    double start, alone, beside;     // tiles: fixed, a key of the longest row with up to 256 tiles, with more
    double full;                     // 32768 keys of a row (a key of a tile on every CU)
};
constexpr Kv4Cost kCost64 = {0.0064, 0.86, 5.5, 0.027, 0.0305, 0.026}, kCost128 = {0.0115, 1.65, 8.7, 0.0455, 0.056, 0.042};

Kv4Plan kv4_plan(int n_heads, int n_kv, int d_head, int T, int ctx_len) {
    Kv4Plan p;
    const long R = (long)T * (n_heads / n_kv), tiles = (R + kTileRows - 1) / kTileRows * n_kv;
    const Kv4Cost& c = d_head == 64 ? kCost64 : kCost128;
    const double pairs = (double)n_heads * T * (ctx_len - 0.5 * (T - 1));
    const double in_blocks = c.block * (double)((R + 15) / 16 * n_kv) + c.pairs * 1e-6 * pairs;
    const double in_tiles = c.start + std::max(ctx_len * (tiles <= 256 ? c.alone : c.beside), c.full * pairs / 32768);
    if (T > 1 && R >= kTileRows && in_tiles < in_blocks) {   // a tile of rows at least: less is mostly none
        p.tiles = true;
        p.blocks = (int)((R + kTileRows - 1) / kTileRows);
        return p;
    }
    const long groups = (ctx_len + kv4::kKeys - 1) / kv4::kKeys;
    auto blocks_of = [&](int rows) {
        p.blocks = (int)((R + rows - 1) / rows);
        p.nch = (int)std::max(1l, std::min((groups + kWaves - 1) / kWaves, kSharers / ((long)p.blocks * n_kv)));
        return (groups + (long)p.nch * kWaves - 1) / ((long)p.nch * kWaves);   // groups of keys of a wave
    };
    const int fewest = 16 / (d_head / 32);
    const long each = blocks_of(fewest);
    p.few = R <= fewest || ((long)p.blocks * n_kv <= kSharers && each <= kFewGroups);
    if (!p.few) {
        blocks_of(16);
        if ((long)p.blocks * n_kv > kSharers && (d_head == 128 || ctx_len <= kFourFrom64)) p.waves = kWaves / 2;
    }
    return p;
}

static_assert(kSharers <= kSmallMaxTiles, "a counter for each block whose keys are shared");
}  // namespace

size_t attn_kv4_part_bytes(int n_heads, int n_kv, int d_head, int T, int ctx_len) {
    // Refused by the launch: no plan, and no scratch that would grow for such a call.
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv || T < 1 || ctx_len < T || (d_head != 64 && d_head != 128)) return 0;
    const Kv4Plan p = kv4_plan(n_heads, n_kv, d_head, T, ctx_len);
    return p.nch > 1 ? (size_t)T * n_heads * p.nch * kv4_part(d_head) * sizeof(float) : 0;
}

int launch_attn_kv4(hipStream_t s, const float* q, const KVLayer& L, int n_heads, int n_kv, int d_head, int max_seq, int T,
                    int ctx_len, float scale, float* out, float* part, int* ctr, const Kv4Model* m) {
    VH_ARG(n_kv >= 1 && n_heads >= 1 && n_heads % n_kv == 0, "attn: n_heads %d not a multiple of n_kv %d", n_heads, n_kv);
    VH_ARG(d_head == 64 || d_head == 128, "attn: d_head %d not in {64,128}", d_head);
    VH_ARG(ctx_len >= 1 && ctx_len <= max_seq && T >= 1 && T <= ctx_len, "attn: %d rows of %d keys in a cache of %d", T,
           ctx_len, max_seq);
    VH_ARG((long)T * n_heads < (1l << 31), "attn: %d rows of %d heads", T, n_heads);
    VH_ARG(!m || (m->ld >= n_heads * d_head && (!m->pos_dev || T == 1)), "attn: bad model call");
    const Kv4Plan p = kv4_plan(n_heads, n_kv, d_head, T, ctx_len);
    VH_ARG(p.blocks <= 65535 && n_kv <= 65535 && (size_t)T * n_heads / n_kv * (n_heads / n_kv) < (1ull << 32),
           "attn: %d rows of %d heads over %d KV heads are beyond a launch", T, n_heads, n_kv);
    VH_ARG(p.nch == 1 || (part && attn_kv4_part_bytes(n_heads, n_kv, d_head, T, ctx_len) < (1ull << 31)), "attn: no scratch");
    Kv4Attn a;
    a.q = q;
    a.kc = reinterpret_cast<const uint8_t*>(L.k);
    a.vc = reinterpret_cast<const uint8_t*>(L.v);
    a.ks = reinterpret_cast<const uint16_t*>(L.ks);
    a.vs = reinterpret_cast<const uint16_t*>(L.vs);
    a.out = out;
    a.part = part;
    const bool merged = ctr && p.nch <= kMergedChunks;
    a.ctr = merged ? ctr : nullptr;
    a.codes = kv4::head_codes(max_seq, d_head);
    a.scales = kv4::head_scales(max_seq, d_head);
    a.n_heads = n_heads;
    a.rep = n_heads / n_kv;
    a.magic = (uint32_t)((1ull << 32) / a.rep + 1);
    a.T = T;
    a.ctx = ctx_len;
    a.ldq = m ? m->ld : n_heads * d_head;
    a.out16 = m ? m->out16 : nullptr;
    a.pos_dev = m ? m->pos_dev : nullptr;
    a.cos_t = m ? m->cos_t : nullptr;
    a.sin_t = m ? m->sin_t : nullptr;
    a.nch = p.nch;
    // Never 0: a masked score's -inf times the factor has to stay -inf.
    a.sl2 = std::max((float)(std::fabs((double)scale) * 1.4426950408889634), 1e-20f);
    a.qsign = scale < 0.f ? -1.f : 1.f;
    if (p.tiles) {
        const dim3 grid(n_kv, p.blocks);
        if (d_head == 64) VH_LAUNCH(kv4_attn_tiles_kernel<64>, grid, dim3(64 * kTileWaves), 0, s, a);
        else VH_LAUNCH(kv4_attn_tiles_kernel<128>, grid, dim3(64 * kTileWaves), 0, s, a);
        VH_LAUNCHED();
        return VLRF_HIP_OK;
    }
    const dim3 grid(p.nch, n_kv, p.blocks);
#define VH_ROWS(D, FEW, W) VH_LAUNCH((kv4_attn_rows_kernel<D, FEW, W>), grid, dim3(64 * W), 0, s, a)
    if (p.few) {
        if (d_head == 64) VH_ROWS(64, true, kWaves);
        else VH_ROWS(128, true, kWaves);
    } else if (p.waves == kWaves / 2) {
        if (d_head == 64) VH_ROWS(64, false, kWaves / 2);
        else VH_ROWS(128, false, kWaves / 2);
    } else {
        if (d_head == 64) VH_ROWS(64, false, kWaves);
        else VH_ROWS(128, false, kWaves);
    }
#undef VH_ROWS
    VH_LAUNCHED();
    if (p.nch == 1 || merged) return VLRF_HIP_OK;
    if (d_head == 64) VH_LAUNCH(kv4_merge_kernel<64>, dim3(T * n_heads), dim3(512), 0, s, part, p.nch, out, a.out16);
    else VH_LAUNCH(kv4_merge_kernel<128>, dim3(T * n_heads), dim3(512), 0, s, part, p.nch, out, a.out16);
    VH_LAUNCHED();
    return VLRF_HIP_OK;
}

}  // namespace vlrf_hip
