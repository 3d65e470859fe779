// kv8.cuh — what the kernels of the 8-bit K/V cache share: the argument blocks, input loads, the RoPE rotation and the
// coding rule (include/flb_kv8.h).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "flb_ptx.cuh"

namespace flb {

// Every kernel of this family is launched with programmatic stream serialisation: its CTAs may become resident while the kernel in front
// drains.  They touch nothing before that kernel, and with it everything before, has completed, and let the next one go after that
// only: for a caller a launch is as ordered as any, it merely starts sooner.  All threads call it first.
// What the kernel in front may write (inputs, lengths, positions) is read by plain loads: the read-only path is for data that nobody writes while a
// kernel is resident, and loads through it may be moved in front of the wait.
__device__ __forceinline__ void kv8_begin() {
    grid_dependency_wait();
    grid_launch_dependents();
}
template <typename Kernel, typename... Args>
inline cudaError_t kv8_launch(Kernel kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

enum : unsigned { kKv8BadLen = 4u, kKv8BadPos = 32u };

struct Kv8Cache {
    int B, H, T;        // H: K/V heads
    int block_shift;    // log2(block_len)
    int nblk;           // blocks per slab
    uint8_t *codes[2];  // K, V
    float *scale[2];
    int *row_pos;
};

struct Kv8Input { // q, k or v rows as the projections leave them
    const void *p;
    const float *w_scale;
    int row_stride;
};

struct Kv8AppendArgs {
    Kv8Cache c;
    int S, nwin; // tokens; blocks that a sequence's tokens can touch
    int max_past; // sequences with more cached rows are left alone
    int start_pos;
    const int *past_lens, *new_lens, *token_pos;
    Kv8Input in[2]; // k, v
    const float *act_scale;
    const float *freq_cis;
    int freq_rows;
    unsigned *status;
};

struct Kv8DecodeArgs {
    Kv8Cache c;
    int input_mode;
    int Hq, G, nchunk; // q heads, q heads per K/V head, CTAs that share a K/V head's q heads out among themselves
    int start_pos;
    const int *past_lens, *token_pos;
    Kv8Input in[3]; // q, k, v
    const float *act_scale;
    const float *freq_cis;
    int freq_rows;
    float scale_log2e, cap_log2e; // softmax_scale, softcap in units of log2
    const float *slopes;
    const int *key_begin;
    float *scores; // [B,Hq,T] log2-domain scores, when weights are accumulated
    float *ml;     // [B,Hq,2] final maximum and sum, likewise
    const float *weight_in;
    float *weight_out;
    void *out;
    int out_f16;
    int append; // the attention kernel stores the new token itself (one CTA per K/V head and split)
    int max_past; // sequences with more cached rows are left alone
    int nsplit_max, split_len;
    unsigned *status, *counters;
    float *part_o, *part_ml;
};

struct Kv8EvictArgs {
    Kv8Cache c;
    int start_pos;
    const int *past_lens;
    int *len_out;
    int budget, recent, sinks;
    const int *next_pos;
    const float *weight;
    float *weight_out;
    int *pos_out;
    unsigned *status;
    int *moves;    // [B*H][T / 2] sources, rising: the kept rows at or behind m, the last of them at the end of its room
    int *holes;    // [B*H][T / 2] holes below m, rising
    int *seq_len;      // [B][2] m, and what becomes of len_out
    float *edge_scale; // [B*H][2] scales of the block that row m lies in, as they were
    int *hole_off; // [B*H][nblk + 1] holes in front of each block
};

cudaError_t launch_kv8_append(const Kv8AppendArgs &a, int d, int code, int input_mode, cudaStream_t stream);
cudaError_t launch_kv8_decode(const Kv8DecodeArgs &a, int d, int code, int nt, cudaStream_t stream);
cudaError_t launch_kv8_evict(const Kv8EvictArgs &a, int d, int code, cudaStream_t stream);

// ---- inputs --------------------------------------------------------------------------------------
// Eight consecutive elements as they lie in memory, and what they stand for.  MODE 0: float(acc) * act_scale * w_scale, in this order; 1: fp32;
// 2: fp16.  Apart, so that a thread can have several loads under way.
struct Kv8Raw {
    uint4 lo, hi; // fp16: lo only
};
template <int MODE> __device__ __forceinline__ Kv8Raw kv8_raw8(const Kv8Input &in, size_t token, int col) {
    const size_t off = token * in.row_stride + col;
    Kv8Raw r;
    if (MODE == 2) {
        r.lo = *reinterpret_cast<const uint4 *>((const __half *)in.p + off);
        r.hi = make_uint4(0u, 0u, 0u, 0u);
    } else {
        const uint4 *p = reinterpret_cast<const uint4 *>((const uint32_t *)in.p + off);
        r.lo = p[0];
        r.hi = p[1];
    }
    return r;
}
template <int MODE> __device__ __forceinline__ void kv8_values8(const Kv8Raw &r, const Kv8Input &in, const float *act_scale, size_t token, int col, float (&x)[8]) {
    if (MODE == 2) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&r.lo);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
        const uint32_t u[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
        if (MODE == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(u[i]);
        } else {
            const float as = act_scale[token];
            const float4 *w = reinterpret_cast<const float4 *>(in.w_scale + col);
            const float4 w0 = w[0], w1 = w[1];
            const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn((float)(int)u[i], as), ws[i]);
        }
    }
}
template <int MODE> __device__ __forceinline__ void kv8_load8(const Kv8Input &in, const float *act_scale, size_t token, int col, float (&x)[8]) {
    kv8_values8<MODE>(kv8_raw8<MODE>(in, token, col), in, act_scale, token, col, x);
}

// Rotation of the pairs (2i, 2i+1) of eight values by a table row (its entries at the same columns).  Every product is
// rounded before the sum, so that the stored codes do not depend on where a compiler fuses.
__device__ __forceinline__ void kv8_rotate8(const float4 &f0, const float4 &f1, float (&x)[8]) {
    const float cs[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float a = x[i], b = x[i + 1];
        // (the packed forms of these would be fused)
        x[i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, cs[i + 1]));
        x[i + 1] = __fadd_rn(__fmul_rn(b, cs[i]), __fmul_rn(a, cs[i + 1]));
    }
}
__device__ __forceinline__ void kv8_rotate8(const float *row, float (&x)[8]) {
    const float4 *f = reinterpret_cast<const float4 *>(row);
    kv8_rotate8(f[0], f[1], x);
}

// table row of a position; one outside the table is flagged and the nearest row taken
__device__ __forceinline__ int kv8_table_row(int pos, int rows, unsigned *status) {
    if (pos >= 0 && pos < rows) return pos;
    if (status) atomicOr(status, kKv8BadPos);
    return pos < 0 ? 0 : rows - 1;
}

// ---- the coding rule -------------------------------------------------------------------------------
constexpr int kCodeI8 = 0, kCodeE4M3 = 1;
template <int CODE> __device__ __forceinline__ constexpr float kv8_top() { return CODE == kCodeI8 ? 127.0f : 448.0f; }

// largest magnitude of eight values and `m`; a NaN stays
__device__ __forceinline__ float kv8_abs_max8(float m, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x[i]), "f"(x[i + 1]));
    return m;
}
// magnitude bits: ordered like the magnitude, NaN above infinity
__device__ __forceinline__ uint32_t kv8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// scale of a block whose incoming rows reach amax (as magnitude bits); `old` = 0 for a block that starts with them
template <int CODE> __device__ __forceinline__ float kv8_new_scale(uint32_t amax_bits, float old) {
    const float need = __fdiv_rn(__uint_as_float(amax_bits), kv8_top<CODE>());
    return (old != old || need <= old) ? old : need; // NaN on either side stays NaN
}

// Four values to four codes: rne, as a byte each.  int8: the addition of 1.5 * 2^23 rounds to a whole number and leaves it in the low byte.
template <int CODE> __device__ __forceinline__ uint32_t kv8_pack4(const float (&y)[4]) {
    if (CODE == kCodeI8) {
        const float2 magic = make_float2(12582912.0f, 12582912.0f);
        const float2 a = __fadd2_rn(make_float2(y[0], y[1]), magic), b = __fadd2_rn(make_float2(y[2], y[3]), magic);
        return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
// Whether among quotients that are off by up to 2^-22 of themselves one could round to another code than the exact one: it lies that near
// to the middle between two codes.
template <int CODE> __device__ __forceinline__ bool kv8_near_tie(const float (&y)[8]) {
    if (CODE == kCodeI8) {
        const float2 magic = make_float2(12582912.0f, 12582912.0f), back = make_float2(-12582912.0f, -12582912.0f);
        float far = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) { // distance to the whole number
            const float2 v = make_float2(y[i], y[i + 1]), w = __fadd2_rn(__fadd2_rn(v, magic), back);
            const float2 d = __ffma2_rn(w, make_float2(-1.0f, -1.0f), v);
            asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(far) : "f"(d.x), "f"(d.y));
        }
        return far > 0.5f - 6.1035156e-5f; // 2^-14 > 127 * 2^-22
    }
    // e4m3 keeps 3 of the 23 mantissa bits (fewer below 2^-6: always looked at exactly there)
    bool near = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(y[i]) & 0x7fffffffu;
        near = near || u < 0x3c800000u || ((u + 8u) & 0xfffffu) - 0x80000u <= 16u;
    }
    return near;
}
// Eight values over their block's scale, rounded to codes; `inv` = 1 / scale.  The quotient is defined as one IEEE division; multiplying by
// the reciprocal is off by 2^-22 at most, which shows only next to a tie, and there the division is done.  A scale of 0, infinity or NaN gives
// codes 0.
// A subnormal scale may be rounded down by up to a third, so the quotients are held to the largest code; a normal one is off by 2^-24 and needs no
// such care.  (out of line: inlined, its eight divisions are issued under a predicate for every value)
template <int CODE> __device__ __forceinline__ float kv8_quotient(float x, float scale) {
    return fminf(fmaxf(__fdiv_rn(x, scale), -kv8_top<CODE>()), kv8_top<CODE>());
}
template <int CODE> __device__ __noinline__ uint2 kv8_encode8_exact(float4 u, float4 v, float scale) {
    const float a[4] = {kv8_quotient<CODE>(u.x, scale), kv8_quotient<CODE>(u.y, scale), kv8_quotient<CODE>(u.z, scale), kv8_quotient<CODE>(u.w, scale)};
    const float b[4] = {kv8_quotient<CODE>(v.x, scale), kv8_quotient<CODE>(v.y, scale), kv8_quotient<CODE>(v.z, scale), kv8_quotient<CODE>(v.w, scale)};
    return make_uint2(kv8_pack4<CODE>(a), kv8_pack4<CODE>(b));
}
template <int CODE> __device__ __forceinline__ uint2 kv8_encode8(const float (&x)[8], float scale, float inv) {
    if (!(scale > 0.f && scale <= 3.402823466e38f)) return make_uint2(0u, 0u);
    const bool exact = !(inv <= 3.402823466e38f && scale <= 1e37f); // the reciprocal of a subnormal scale overflows, that of a huge one is subnormal
    float y[8];
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 v = __fmul2_rn(make_float2(x[i], x[i + 1]), inv2);
        y[i] = v.x;
        y[i + 1] = v.y;
    }
    if (exact || kv8_near_tie<CODE>(y)) return kv8_encode8_exact<CODE>(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), scale);
    const float a[4] = {y[0], y[1], y[2], y[3]}, b[4] = {y[4], y[5], y[6], y[7]};
    return make_uint2(kv8_pack4<CODE>(a), kv8_pack4<CODE>(b));
}
// what eight codes stand for, before the scale
template <int CODE> __device__ __forceinline__ void kv8_decode8(uint2 u, float (&x)[8]) {
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (CODE == kCodeI8) { // byte + 128 under the exponent of 2^23
            const uint32_t v = w[j] ^ 0x80808080u;
            const float2 back = make_float2(-8388736.0f, -8388736.0f);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float2 f = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(v, 0x4b000000u, 0x7440 + i)), __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7441 + i))), back);
                x[4 * j + i] = f.x;
                x[4 * j + i + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[j] >> (16 * i)), __NV_E4M3);
                const float2 f = __half22float2(__half2(h));
                x[4 * j + 2 * i] = f.x;
                x[4 * j + 2 * i + 1] = f.y;
            }
        }
    }
}
__device__ __forceinline__ void kv8_scale8(float (&x)[8], float s) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 v = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(s, s));
        x[i] = v.x;
        x[i + 1] = v.y;
    }
}
// codes of a block that a larger scale takes over: ratio = old / new
template <int CODE> __device__ __forceinline__ uint2 kv8_rescale8(uint2 u, float ratio) {
    float x[8];
    kv8_decode8<CODE>(u, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], ratio); // rounded, then rounded to a code: not to be fused with the packing's addition
    const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
    return make_uint2(kv8_pack4<CODE>(a), kv8_pack4<CODE>(b));
}

// largest of a value over the block's threads; `red` has room for one word per warp.  All threads call it.
__device__ __forceinline__ uint32_t kv8_block_max(uint32_t v, uint32_t *red) {
    v = __reduce_max_sync(0xffffffffu, v);
    const int nw = (blockDim.x + 31) >> 5;
    if (nw == 1) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = ((int)(threadIdx.x & 31) < nw) ? red[threadIdx.x & 31] : 0u;
    v = __reduce_max_sync(0xffffffffu, v);
    return v;
}

} // namespace flb
