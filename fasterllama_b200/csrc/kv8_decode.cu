// kv8_decode.cu — single-token attention over the 8-bit cache, the new token's append included.
//
// For one K/V head and its G q heads:  x_r = c q.(code_r scale_r),  out = sum_r p_r code_r scale_r / sum_r p_r.
// HBM-bound: 2 d bytes per cached row and K/V head, read once for all G heads.  16 x 32 heads of 1024-2047 rows: 43-45 us, 4.5-4.8 TB/s (41-42
// us from a replayed graph); batches of 16, 32, 48 x 1535 rows take 40, 68, 98 us: 11 us (launch, ramp, drain, joining) + bytes / 7.0 TB/s.
//   * grid = K/V heads x splits of `split_len` rows; four warps per CTA, warp w takes the 16-row steps w, w + 4, ... of its
//     split.  Every warp copies its own steps (cp.async, 16 bytes a lane) into a ring of its own in shared memory, three and more
//     steps ahead: 192 KB per SM under way, no barrier between warps.  The first copies leave before q is looked at.
//     16-byte chunks are permuted within the rows so that both products' fragment loads are free of bank conflicts.
//   * both products run on the warp-level matrix instructions with exact operands, the columns being parts of q or p:
//     S = K q, int8:  A = 16 rows of codes as they are, B = q as a 28-bit whole number in four base-128 digits (two tiles of four
//                     heads); the int32 sums are exact, no code is converted
//     S = K q, e4m3:  A = codes as fp16 (exact), B = q in a high and a low fp16 part, 22 bits
//     O^T += V^T p:   A = codes of 16 dims x 16 rows as fp16 (two rows' bytes interleaved; 1.5 instructions per code), B = p in two
//                     fp16 parts, an 8x8 transpose away from S.  Floating parts keep small weights exact too, digits would not.
//     Lane (g, t) ends with rows g, g + 8 of head t, both parts in its own registers.
//   * scales of a block are uniform over a step (blocks hold at least 16 rows): K's goes into the score, V's into p.
//   * each warp keeps its own running maximum per head, raised only when a score passes it by 2^8 (exact: sum and result
//     share the reference); warps merge in warp order, splits in split order by the CTA that arrives last.  The
//     result depends on the sequence and on split_len alone.
//   * the CTA of the last split codes the new token and rescales its block if that has to grow, before it reads it; no
//     other CTA reads that block (splits are multiples of blocks).  Where several CTAs share a K/V head (more q heads than
//     fit one), the append kernel runs first instead.
//   * weights for an eviction need the final maximum and sum: scores are left in scratch (fp32) and a second small kernel turns
//     them into weights and adds them up over the group.
#include "kv8.cuh"

#include <atomic>
#include <climits>

namespace flb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -1e30f;   // running maximum before the first visible key (finite: -inf - -inf is NaN)
constexpr float kRaise = 8.0f;     // log2: a weight stays below 2^8
constexpr int kWarps = 4;
constexpr int kStep = 16;          // rows per warp step

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// Two codes (bytes i0, i1 of w) as an fp16 pair.  int8: byte + 128 under the exponent of 1024, minus 1152.
template <int CODE> __device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (CODE == kCodeI8) {
        w ^= 0x80808080u;
        const uint32_t bias = 0x64806480u;
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        lo = h2_bits(__hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<const __half2 *>(&bias)));
        hi = h2_bits(__hsub2(*reinterpret_cast<__half2 *>(&b), *reinterpret_cast<const __half2 *>(&bias)));
    } else {
        lo = h2_bits(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
        hi = h2_bits(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
    }
}

// ---- a warp's ring: one slot holds 16 rows of K codes, then 16 rows of V codes
template <int D> struct Ring {
    static constexpr int kRowsBytes = kStep * D;
    static constexpr int kSlot = 2 * kRowsBytes;
    static constexpr int kStages = D == 64 ? 6 : D == 128 ? 3 : 2; // 12 KB per warp (d = 256: 16 KB)
    static constexpr int kWarpBytes = kStages * kSlot;
    // Where chunk c (16 bytes) of row r lies.  K is read as rows r, r + 1 x four neighbouring chunks per eight lanes, V as rows r, r + 2, r + 4,
    // r + 6 x two neighbouring chunks: the permutations send both to eight different chunks of the 128-byte bank line.
    static __device__ __forceinline__ int at(int r, int c) {
        if (D == 64) return (r >> 1) * 128 + ((((r >> 1) ^ r) & 1) << 6) + ((c ^ ((r >> 1) & 2)) << 4);
        return r * D + ((c ^ ((r & 6) ^ ((r & 1) << 2))) << 4);
    }
};
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A store whose line is to outlive the streamed codes in L2: the weights kernel reads it back.
__device__ __forceinline__ uint64_t keep_policy() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void store_kept(float *p, float x, uint64_t policy) {
    asm volatile("st.global.L2::cache_hint.f32 [%0], %1, %2;" ::"l"(p), "f"(x), "l"(policy) : "memory");
}

// 16 rows from `k` and `v` into a slot
template <int D> __device__ __forceinline__ void copy_step(uint32_t slot, const uint8_t *k, const uint8_t *v, int lane) {
    constexpr int CPR = D / 16, PER = kStep * CPR / 32;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int id = lane + 32 * i, r = id / CPR, c = id % CPR;
        const int to = Ring<D>::at(r, c);
        copy16(slot + to, k + id * 16);
        copy16(slot + Ring<D>::kRowsBytes + to, v + id * 16);
    }
}

// a few rows per CTA: the input form is looked at here and not compiled in
__device__ __forceinline__ void load8(const Kv8DecodeArgs &a, int which, size_t token, int col, float (&x)[8]) {
    if (a.input_mode == 0)
        kv8_load8<0>(a.in[which], a.act_scale, token, col, x);
    else if (a.input_mode == 1)
        kv8_load8<1>(a.in[which], a.act_scale, token, col, x);
    else
        kv8_load8<2>(a.in[which], a.act_scale, token, col, x);
}

// What the new token does to its block, K and V: the block's scale from now on, and what the codes it held are to be multiplied by.
struct TokenScales {
    float scale[2], ratio[2];
    int grown[2];
};
// Stores k (kv = 0) or v of the new token, by one warp; lane i has eight dims.
template <int D, int CODE>
__device__ __forceinline__ void append_token(const Kv8DecodeArgs &a, int kv, size_t unit, int b, int h, int past, int pos, int prow, TokenScales *ts) {
    const int lane = threadIdx.x & 31, blk = past >> a.c.block_shift;
    const size_t sidx = unit * a.c.nblk + blk;
    const float old = (blk << a.c.block_shift) == past ? 0.f : a.c.scale[kv][sidx];
    float x[8];
    uint32_t amax = 0;
    if (lane < D / 8) {
        load8(a, 1 + kv, (size_t)b, h * D + lane * 8, x);
        if (kv == 0 && a.freq_cis) kv8_rotate8(a.freq_cis + (size_t)prow * D + lane * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, kv8_abs_bits(x[e]));
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    const float scale = kv8_new_scale<CODE>(amax, old);
    if (lane < D / 8) *reinterpret_cast<uint2 *>(a.c.codes[kv] + (unit * a.c.T + past) * D + lane * 8) = kv8_encode8<CODE>(x, scale, __fdiv_rn(1.f, scale));
    if (lane == 0) {
        a.c.scale[kv][sidx] = scale;
        if (kv == 0 && a.c.row_pos) a.c.row_pos[unit * a.c.T + past] = pos;
        const bool grown = old > 0.f && scale > old;
        ts->scale[kv] = scale;
        ts->grown[kv] = grown;
        ts->ratio[kv] = grown ? __fdiv_rn(old, scale) : 1.f;
    }
}

// head dimension of column p of an accumulator row (see the output products: tile i, lane group g, half e)
template <int D> __device__ __forceinline__ int dim_of(int p) {
    const int i = p >> 4, g = (p & 15) >> 1;
    return (i >> 3) * 128 + g * (D == 64 ? 8 : 16) + 2 * (i & 7) + (p & 1);
}

// FORM: capped scores, distance bias or key_begin.  NT: column tiles of eight = four q heads each.
template <int D, int CODE, int NT, bool FORM>
__global__ void __launch_bounds__(kWarps * 32, D == 128 ? (NT == 1 ? 4 : 3) : 1) flb_kv8_decode_kernel(const __grid_constant__ Kv8DecodeArgs a) {
    constexpr int HEADS = 4 * NT;
    constexpr int KCH = D / 64;   // 16-byte chunks of a K row per lane
    constexpr int VW = D / 32;    // 32-bit words of a V row per lane
    constexpr int MT = D / 16;    // output tiles of 16 dims
    constexpr int NTHREADS = kWarps * 32;
    constexpr int QH = HEADS / kWarps; // q heads that a warp prepares
    __shared__ __align__(16) unsigned char q_s[HEADS * D * 4]; // e4m3: fp16 [2 head + part][D]; int8: bytes [part][head][D]
    __shared__ float q_unit[HEADS];                        // what a product with q_s is to be multiplied by
    __shared__ float w_m[kWarps][HEADS], w_l[kWarps][HEADS];
    extern __shared__ __align__(128) unsigned char ring_smem[];
    // The warps' results, in the rings' room once they are through.  Dims in the order in which the accumulators hold them (column 16 i + 2 g + e is
    // dim_of() that) and 16 words between heads: the stores of a warp then meet no bank twice more than they have to.
    float(*w_o)[HEADS][D + 16] = reinterpret_cast<float(*)[HEADS][D + 16]>(ring_smem);
    __shared__ TokenScales ts;
    __shared__ int last_flag;

    kv8_begin();
    const int split = (int)(blockIdx.x % (unsigned)a.nsplit_max);
    const unsigned uc = blockIdx.x / (unsigned)a.nsplit_max;
    const int chunk = (int)(uc % (unsigned)a.nchunk);
    const size_t unit = uc / (unsigned)a.nchunk;
    const int b = (int)(unit / a.c.H), h = (int)(unit - (size_t)b * a.c.H);
    const int head0 = h * a.G + chunk * HEADS, nheads = min(HEADS, a.G - chunk * HEADS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    const int past = a.past_lens ? a.past_lens[b] : a.start_pos;
    const int pos = a.token_pos ? a.token_pos[b] : past;
    float qx[QH][8];
    static_assert(D <= 256, "a warp holds a row, eight dims to a lane");
#pragma unroll
    for (int i = 0; i < QH; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) qx[i][e] = 0.f;
        if (warp + i * kWarps < nheads && lane < D / 8) load8(a, 0, (size_t)b, (head0 + warp + i * kWarps) * D + lane * 8, qx[i]);
    }
    if (past < 0 || past > a.max_past) { // flagged, nothing stored, zeros returned
        if (split == 0) {
            if (tid == 0) atomicOr(a.status, kKv8BadLen);
            for (int i = tid; i < nheads * D; i += NTHREADS) {
                const size_t o = ((size_t)b * a.Hq + head0) * D + i;
                if (a.out_f16) ((__half *)a.out)[o] = __float2half_rn(0.f); else ((float *)a.out)[o] = 0.f;
            }
        }
        return;
    }
    const int nsplit = past / a.split_len + 1;
    if (split >= nsplit) return;
    const int row0 = split * a.split_len, row1 = min(row0 + a.split_len, past + 1);
    const bool is_last = split == nsplit - 1;
    const int prow = a.freq_cis ? kv8_table_row(pos, a.freq_rows, a.status) : 0;
    const int begin = (FORM && a.key_begin) ? a.key_begin[b] : INT_MIN;

    // ---- the warp's steps: rows r, r + 64, ...
    using R = Ring<D>;
    constexpr int kStride = kWarps * kStep;
    int r = row0 + warp * kStep;
    // rows in position order: nothing below key_begin is read
    if (FORM && a.key_begin && !a.c.row_pos && begin > r) r += (int)(((long long)min(begin, a.c.T) - r) / kStride) * kStride;
    const uint32_t ring = smem_u32(ring_smem) + (uint32_t)(warp * R::kWarpBytes);
    const uint8_t *ksrc = a.c.codes[0] + (unit * a.c.T + r) * (size_t)D, *vsrc = a.c.codes[1] + (unit * a.c.T + r) * (size_t)D;
    int fetch = r, fslot = 0; // next step to copy, and its slot
    auto copy_next = [&](int end) {
        if (fetch < end) {
            copy_step<D>(ring + fslot * R::kSlot, ksrc, vsrc, lane);
            ksrc += (size_t)kStride * D;
            vsrc += (size_t)kStride * D;
            fetch += kStride;
            fslot = fslot + 1 == R::kStages ? 0 : fslot + 1;
        }
    };
    // Everything but the block that the new token goes into can be on its way at once.
    const bool storing = is_last && a.append;
    const int settled = storing ? min(row1, past >> a.c.block_shift << a.c.block_shift) : row1;
    int groups = 0;
#pragma unroll
    for (int i = 0; i < R::kStages; ++i)
        if (fetch < settled) {
            copy_next(settled);
            copy_commit();
            ++groups;
        }
    // scales of the warp's steps: lane i has those of step i
    float sc_k = 0.f, sc_v = 0.f;
    const int sblk = (r + lane * kStride) >> a.c.block_shift;
    if (r + lane * kStride < settled) {
        sc_k = __ldcg(a.c.scale[0] + unit * a.c.nblk + sblk);
        sc_v = __ldcg(a.c.scale[1] + unit * a.c.nblk + sblk);
    }
    if (storing && warp >= 2) append_token<D, CODE>(a, warp - 2, unit, b, h, past, pos, prow, &ts);

    // ---- q: rotated, brought to a fixed range by a power of two, cut into parts; one warp per head
#pragma unroll
    for (int i = 0; i < QH; ++i) {
        const int hh = warp + i * kWarps;
        uint32_t amax = 0;
        if (hh < nheads && lane < D / 8 && a.freq_cis) kv8_rotate8(a.freq_cis + (size_t)prow * D + lane * 8, qx[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, kv8_abs_bits(qx[i][e]));
        amax = __reduce_max_sync(0xffffffffu, amax);
        // int8: |q| < 2^27 as a whole number in four signed base-128 digits; e4m3: |q| < 2^9 in two fp16 parts
        constexpr int kTop = CODE == kCodeI8 ? 26 : 8;
        const int ex = min(max((int)(amax >> 23) - 127, -100), 126);
        const float up = __uint_as_float((uint32_t)(kTop - ex + 127) << 23), down = __uint_as_float((uint32_t)(ex - kTop + 127) << 23);
        if (lane < D / 8) {
            if (CODE == kCodeI8) {
                uint32_t dig[4][2] = {};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int v = __float2int_rn(qx[i][e] * up);
                    const int sh = 8 * (e & 3);
                    dig[0][e >> 2] |= (uint32_t)((v >> 21) & 0xff) << sh; // -64..64
                    dig[1][e >> 2] |= (uint32_t)((v >> 14) & 0x7f) << sh;
                    dig[2][e >> 2] |= (uint32_t)((v >> 7) & 0x7f) << sh;
                    dig[3][e >> 2] |= (uint32_t)(v & 0x7f) << sh;
                }
#pragma unroll
                for (int p = 0; p < 4; ++p) *reinterpret_cast<uint2 *>(q_s + (p * HEADS + hh) * D + lane * 8) = make_uint2(dig[p][0], dig[p][1]);
            } else {
                __half2 hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float u = qx[i][2 * e] * up, v = qx[i][2 * e + 1] * up;
                    hi[e] = __floats2half2_rn(u, v);
                    const float2 f = __half22float2(hi[e]);
                    lo[e] = __floats2half2_rn(u - f.x, v - f.y);
                }
                *reinterpret_cast<uint4 *>(q_s + (2 * hh * D + lane * 8) * 2) = *reinterpret_cast<uint4 *>(hi);
                *reinterpret_cast<uint4 *>(q_s + ((2 * hh + 1) * D + lane * 8) * 2) = *reinterpret_cast<uint4 *>(lo);
            }
        }
        // an infinite or NaN q makes its scores NaN
        if (lane == 0) q_unit[hh] = amax < 0x7f800000u ? down * a.scale_log2e : __uint_as_float(0x7fffffffu);
    }
    __syncthreads();
    if (storing) {
        if (ts.grown[0] || ts.grown[1]) { // the codes that the block held follow its scale
            const int blk0 = past >> a.c.block_shift << a.c.block_shift;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint2 *rows = reinterpret_cast<uint2 *>(a.c.codes[i] + (unit * a.c.T + blk0) * D);
                if (ts.grown[i])
                    for (int c = tid; c < (past - blk0) * (D / 8); c += NTHREADS) rows[c] = kv8_rescale8<CODE>(rows[c], ts.ratio[i]);
            }
            __syncthreads();
        }
        if (r + lane * kStride >= settled) { // steps of that block
            sc_k = ts.scale[0];
            sc_v = ts.scale[1];
        }
    }
    for (; groups < R::kStages; ++groups) { // a group per stage, empty where there is no step
        copy_next(row1);
        copy_commit();
    }
    // The largest V scale decides by which power of two the weights are raised before they are cut into fp16 parts.  Steps that hold no visible row
    // have no say: a scale there may be anything, an infinity or NaN included.
    bool seen = r + lane * kStride < row1;
    if (FORM && a.key_begin && seen) {
        const int s0 = r + lane * kStride, s1 = min(s0 + kStep, row1);
        if (a.c.row_pos) {
            int newest = INT_MIN;
#pragma unroll 4
            for (int s = s0; s < s1; ++s) newest = max(newest, __ldcg(a.c.row_pos + unit * a.c.T + s));
            seen = newest >= begin;
        } else {
            seen = s1 > begin;
        }
    }
    const uint32_t vmax = __reduce_max_sync(0xffffffffu, seen ? kv8_abs_bits(sc_v) : 0u);
    const int vex = min(max((int)(vmax >> 23) - 127, -121), 126); // both powers of two below stay normal numbers
    const float v_up = __uint_as_float((uint32_t)(5 - vex + 127) << 23), v_down = __uint_as_float((uint32_t)(vex - 5 + 127) << 23);

    // q as the matrix instructions take it.  Lane (g, t) meets dims 64 c + 16 t .. + 15 of a row; column 2 t + i of a tile is part i (int8: of the second
    // tile part 2 + i) of head t
    constexpr int QT = CODE == kCodeI8 ? 2 : 1, QS = CODE == kCodeI8 ? 2 * KCH : 4 * KCH;
    uint32_t qf[NT][QT][QS][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int p = 0; p < QT; ++p)
#pragma unroll
            for (int st = 0; st < QS; ++st) {
                const unsigned char *src = CODE == kCodeI8 ? q_s + ((2 * p + (g & 1)) * HEADS + 4 * n + (g >> 1)) * D + (st >> 1) * 64 + 16 * t + 8 * (st & 1)
                                                           : q_s + ((8 * n + g) * D + (st >> 2) * 64 + 16 * t + 4 * (st & 3)) * 2;
                const uint2 u = *reinterpret_cast<const uint2 *>(src);
                qf[n][p][st][0] = u.x;
                qf[n][p][st][1] = u.y;
            }
    float qu[NT], m_run[NT], l_run[NT], slope[NT];
    float o[NT][MT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        qu[n] = q_unit[4 * n + t];
        m_run[n] = kNoMax;
        l_run[n] = 0.f;
        slope[n] = (FORM && a.slopes && 4 * n + t < nheads) ? a.slopes[head0 + 4 * n + t] * kLog2e : 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    }
    const float inv_cap = (FORM && a.cap_log2e > 0.f) ? 1.0f / a.cap_log2e : 0.f;

    // ---- the pass over the rows
    // This lane's reads of a slot: K rows g, g + 8 (the rows of a step's tile are dealt out so that eight lanes meet eight chunks), V rows
    // 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    const uint64_t keep = a.scores ? keep_policy() : 0ull;
    int slot = 0, step = 0;
    for (; r < row1; r += kStride) {
        copy_wait<R::kStages - 1>();
        __syncwarp();
        const unsigned char *ks_p = ring_smem + warp * R::kWarpBytes + slot * R::kSlot, *vs_p = ks_p + R::kRowsBytes;
        float x[NT][2]; // scores of rows g, g + 8 by head, as products of codes
        {
            float sf[NT][4];
            int si[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sf[n][e] = 0.f;
                    si[n][0][e] = si[n][1][e] = 0;
                }
#pragma unroll
            for (int c = 0; c < KCH; ++c) {
                const uint4 k0 = *reinterpret_cast<const uint4 *>(ks_p + R::at(g, 4 * c + t));
                const uint4 k1 = *reinterpret_cast<const uint4 *>(ks_p + R::at(g + 8, 4 * c + t));
                const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
                if (CODE == kCodeI8) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint32_t f[4] = {w0[2 * w], w1[2 * w], w0[2 * w + 1], w1[2 * w + 1]};
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int p = 0; p < 2; ++p) mma16832(si[n][p], f, qf[n][p % QT][2 * c + w][0], qf[n][p % QT][2 * c + w][1]);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t f[4];
                        codes_to_halves<CODE>(w0[w], f[0], f[2]);
                        codes_to_halves<CODE>(w1[w], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816(sf[n], f, qf[n][0][(4 * c + w) % QS][0], qf[n][0][(4 * c + w) % QS][1]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    x[n][i] = CODE == kCodeI8 ? fmaf((float)(si[n][0][2 * i] * 128 + si[n][0][2 * i + 1]), 16384.0f, (float)(si[n][1][2 * i] * 128 + si[n][1][2 * i + 1]))
                                              : sf[n][2 * i] + sf[n][2 * i + 1];
        }
        const float ks = __shfl_sync(0xffffffffu, sc_k, step), vs = __shfl_sync(0xffffffffu, sc_v, step) * v_up;
        ++step;
        int kpos[2] = {r + g, r + g + 8};
        bool vis[2] = {true, true};
        if (r + kStep > row1) {
            vis[0] = r + g < row1;
            vis[1] = r + g + 8 < row1;
        }
        if (FORM) {
            if (a.c.row_pos && (a.slopes || a.key_begin)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) kpos[i] = __ldcg(a.c.row_pos + unit * a.c.T + r + g + 8 * i);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) vis[i] = vis[i] && kpos[i] >= begin;
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) x[n][i] *= ks * qu[n];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (FORM && a.cap_log2e > 0.f) x[n][i] = cap_score(x[n][i], a.cap_log2e, inv_cap);
                if (FORM) x[n][i] = fmaf(-slope[n], (float)__sad(pos, kpos[i], 0u), x[n][i]);
                x[n][i] = vis[i] ? x[n][i] : -INFINITY;
            }
            if (a.scores && 4 * n + t < nheads) {
                float *sp = a.scores + ((size_t)b * a.Hq + head0 + 4 * n + t) * a.c.T + r + g;
                if (r + g < row1) store_kept(sp, x[n][0], keep);
                if (r + g + 8 < row1) store_kept(sp + 8, x[n][1], keep);
            }
            const float top = fmaxf(x[n][0], x[n][1]);
            if (__any_sync(0xffffffffu, top > m_run[n] + kRaise)) {
                float mx = top;
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float m_new = fmaxf(m_run[n], mx);
                const float corr = ex2(m_run[n] - m_new);
                m_run[n] = m_new;
                l_run[n] *= corr;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] *= corr;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float p = ex2(x[n][i] - m_run[n]);
                l_run[n] += p;
                const float pv = vis[i] ? p * vs : 0.f;
                const __half hi = __float2half_rn(pv);
                const __half lo = __float2half_rn(pv - __half2float(hi));
                pb[n][i] = transpose8x8(h2_bits(__halves2half2(hi, lo)));
            }
        }
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int vr = 2 * t + (i & 1) + (i >> 1) * 8;
            if (D == 64) {
                const uint2 u = *reinterpret_cast<const uint2 *>(vs_p + R::at(vr, g >> 1) + (g & 1) * 8);
                v[i][0] = u.x;
                v[i][1] = u.y;
            } else {
#pragma unroll
                for (int j = 0; j < VW / 4; ++j) { // dims 16 g .. (d = 256: and 128 + 16 g ..)
                    const uint4 u = *reinterpret_cast<const uint4 *>(vs_p + R::at(vr, g + 8 * j));
                    v[i][4 * j] = u.x;
                    v[i][4 * j + 1] = u.y;
                    v[i][4 * j + 2] = u.z;
                    v[i][4 * j + 3] = u.w;
                }
            }
            if (CODE == kCodeE4M3 && r + vr >= row1) // codes behind the sequence may be NaN patterns
#pragma unroll
                for (int w = 0; w < VW; ++w) v[i][w] = 0u;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) { // four dims: two output tiles
            uint32_t f0[4], f1[4];
            const uint32_t e0 = __byte_perm(v[0][w], v[1][w], 0x5140), e1 = __byte_perm(v[0][w], v[1][w], 0x7362);
            const uint32_t e2 = __byte_perm(v[2][w], v[3][w], 0x5140), e3 = __byte_perm(v[2][w], v[3][w], 0x7362);
            codes_to_halves<CODE>(e0, f0[0], f0[1]);
            codes_to_halves<CODE>(e2, f0[2], f0[3]);
            codes_to_halves<CODE>(e1, f1[0], f1[1]);
            codes_to_halves<CODE>(e3, f1[2], f1[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma16816(o[n][2 * w], f0, pb[n][0], pb[n][1]);
                mma16816(o[n][2 * w + 1], f1, pb[n][0], pb[n][1]);
            }
        }
        __syncwarp(); // the slot has been read
        copy_next(row1);
        copy_commit();
        slot = slot + 1 == R::kStages ? 0 : slot + 1;
    }
    copy_wait<0>();
    __syncthreads(); // the rings' room is free

    // ---- warps to shared memory: sums over the eight row groups, high and low parts together
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l_run[n] += __shfl_xor_sync(0xffffffffu, l_run[n], off);
        if (g == 0) {
            w_m[warp][4 * n + t] = m_run[n];
            w_l[warp][4 * n + t] = l_run[n];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
            *reinterpret_cast<float2 *>(&w_o[warp][4 * n + t][16 * i + 2 * g]) =
                make_float2((o[n][i][0] + o[n][i][1]) * v_down, (o[n][i][2] + o[n][i][3]) * v_down);
    }
    __syncthreads();

    // two finished values of a head, at dims d, d + 1
    auto put = [&](int hh, int dim, float y0, float y1) {
        const size_t oo = ((size_t)b * a.Hq + head0 + hh) * D + dim;
        if (a.out_f16)
            *reinterpret_cast<__half2 *>((__half *)a.out + oo) = __floats2half2_rn(y0, y1);
        else
            *reinterpret_cast<float2 *>((float *)a.out + oo) = make_float2(y0, y1);
    };
    auto finish = [&](int hh, int quad, const float4 &acc, float M, float l) { // columns 4 quad ..: two pairs of dims
        const float inv = (l > 0.f || l != l) ? 1.0f / l : 0.f;
        put(hh, dim_of<D>(4 * quad), acc.x * inv, acc.y * inv);
        put(hh, dim_of<D>(4 * quad + 2), acc.z * inv, acc.w * inv);
        if (a.ml && quad == 0) *reinterpret_cast<float2 *>(a.ml + ((size_t)b * a.Hq + head0 + hh) * 2) = make_float2(M, l);
    };

    // ---- merge in warp order, four columns to a thread
    const size_t pbase = ((unit * a.nchunk + chunk) * a.nsplit_max + split) * HEADS;
    for (int i = tid; i < nheads * (D / 4); i += NTHREADS) {
        const int hh = i / (D / 4), quad = i % (D / 4);
        float M = kNoMax, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, w_m[w][hh]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float e = ex2(w_m[w][hh] - M);
            const float4 v = *reinterpret_cast<const float4 *>(&w_o[w][hh][4 * quad]);
            acc.x = fmaf(v.x, e, acc.x);
            acc.y = fmaf(v.y, e, acc.y);
            acc.z = fmaf(v.z, e, acc.z);
            acc.w = fmaf(v.w, e, acc.w);
            l = fmaf(w_l[w][hh], e, l);
        }
        if (nsplit == 1) {
            finish(hh, quad, acc, M, l);
        } else {
            reinterpret_cast<float4 *>(a.part_o)[(pbase + hh) * (D / 4) + quad] = acc;
            if (quad == 0) reinterpret_cast<float2 *>(a.part_ml)[pbase + hh] = make_float2(M, l);
        }
    }
    if (nsplit == 1) return;
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        const unsigned old = atomicAdd(a.counters + unit * a.nchunk + chunk, 1u);
        last_flag = old == (unsigned)(nsplit - 1);
    }
    __syncthreads();
    if (!last_flag) return;
    __threadfence();
    // The last split joins all: maximum and sum per head by a warp, then every thread four columns of one head over its share of the
    // splits, sixteen loads under way, weights of 64 splits at a time in shared memory; the shares are added up in order.
    const size_t mbase = (unit * a.nchunk + chunk) * a.nsplit_max;
    float *const e_s = reinterpret_cast<float *>(ring_smem) + NTHREADS * 4; // [64][HEADS] behind the shares
    for (int hh = warp; hh < nheads; hh += kWarps) {
        const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + mbase * HEADS + hh;
        // the first 64 splits stay in registers: their weights need no second look
        const float2 own = lane < nsplit ? __ldcg(ml + (size_t)lane * HEADS) : make_float2(kNoMax, 0.f);
        const float2 own2 = lane + 32 < nsplit ? __ldcg(ml + (size_t)(lane + 32) * HEADS) : make_float2(kNoMax, 0.f);
        float M = fmaxf(own.x, own2.x);
        for (int s = lane + 64; s < nsplit; s += 32) M = fmaxf(M, __ldcg(ml + (size_t)s * HEADS).x);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
        const float e0 = ex2(own.x - M), e1 = ex2(own2.x - M);
        e_s[lane * HEADS + hh] = e0;
        e_s[(lane + 32) * HEADS + hh] = e1;
        float l = fmaf(own2.y, e1, own.y * e0);
        for (int s = lane + 64; s < nsplit; s += 32) {
            const float2 v = __ldcg(ml + (size_t)s * HEADS);
            l = fmaf(v.y, ex2(v.x - M), l);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        if (lane == 0) {
            w_m[0][hh] = M;
            w_l[0][hh] = l;
        }
    }
    __syncthreads();
    const int quads = nheads * (D / 4), shares = max(1, NTHREADS / quads);
    for (int q0 = 0; q0 < quads; q0 += NTHREADS) {
        const int quad = shares > 1 ? tid % quads : q0 + tid, share = shares > 1 ? tid / quads : 0;
        const bool on = quad < quads && share < shares;
        const int hh = on ? quad / (D / 4) : 0;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 *po = reinterpret_cast<const float4 *>(a.part_o) + mbase * HEADS * (D / 4) + quad;
        for (int s0 = 0; s0 < nsplit; s0 += 64) {
            const int ns = min(64, nsplit - s0);
            if (nsplit > 64 && (q0 > 0 || s0 > 0)) { // (the first 64 are there)
                __syncthreads();
                for (int i = tid; i < ns * nheads; i += NTHREADS) {
                    const int s = i / nheads, hd = i - s * nheads;
                    e_s[s * HEADS + hd] = ex2(__ldcg(a.part_ml + ((mbase + s0 + s) * HEADS + hd) * 2) - w_m[0][hd]);
                }
                __syncthreads();
            }
            if (!on) continue;
#pragma unroll 16
            for (int s = share; s < ns; s += shares) {
                const float4 v = __ldcg(po + (size_t)(s0 + s) * HEADS * (D / 4));
                const float e = e_s[s * HEADS + hh];
                acc.x = fmaf(v.x, e, acc.x);
                acc.y = fmaf(v.y, e, acc.y);
                acc.z = fmaf(v.z, e, acc.z);
                acc.w = fmaf(v.w, e, acc.w);
            }
        }
        if (shares > 1) {
            float4 *sum = reinterpret_cast<float4 *>(ring_smem);
            sum[tid] = acc;
            __syncthreads();
            if (on && share == 0)
                for (int j = 1; j < shares; ++j) {
                    const float4 v = sum[j * quads + quad];
                    acc.x += v.x;
                    acc.y += v.y;
                    acc.z += v.z;
                    acc.w += v.w;
                }
        }
        if (on && share == 0) finish(hh, quad - hh * (D / 4), acc, w_m[0][hh], w_l[0][hh]);
    }
    if (tid == 0) a.counters[unit * a.nchunk + chunk] = 0u; // ready for the next call
}

constexpr int kHeadsAtOnce = 8;

// weight_out = weight_in + sum over the group of 2^(score - max) / sum.  A thread takes four rows of one K/V head; HBM-bound, 4 (G + 2) bytes a
// row and head (100001 rows, 8 heads of 4 q heads, scores from L2: 7.6 us, 1.2 TB/s of scores and weights; latency).
__global__ void __launch_bounds__(256) flb_kv8_weights_kernel(const __grid_constant__ Kv8DecodeArgs a, int blocks_per_unit) {
    const size_t unit = blockIdx.x / (unsigned)blocks_per_unit;
    const int r = ((int)(blockIdx.x % (unsigned)blocks_per_unit) * 256 + threadIdx.x) * 4;
    const int b = (int)(unit / a.c.H), h = (int)(unit - (size_t)b * a.c.H);
    // The kernel in front is the attention kernel, which lets this one start only after everything before it has completed, and writes neither
    // lengths nor weights: they are read while it runs (from L2: this SM's L1 may be older than what came before).
    const int past = a.past_lens ? __ldcg(a.past_lens + b) : a.start_pos;
    const bool on = past >= 0 && past <= a.max_past && r <= past;
    const size_t i = unit * a.c.T + r; // T is a multiple of 16: four rows never leave the slab
    const int begin = a.key_begin && !a.c.row_pos ? __ldcg(a.key_begin + b) : INT_MIN; // no score was left below it
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (on) {
        const float4 in = __ldcg(reinterpret_cast<const float4 *>(a.weight_in + i));
        w[0] = in.x;
        w[1] = in.y;
        w[2] = in.z;
        w[3] = in.w;
    }
    __shared__ float2 ml_s[kHeadsAtOnce];
    kv8_begin();
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r + e == past) w[e] = 0.f;
    const size_t hq0 = (size_t)b * a.Hq + h * a.G;
    const float *scores = a.scores + hq0 * a.c.T + r;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ml) + hq0;
    float sum[4] = {0.f, 0.f, 0.f, 0.f}; // over the group, apart from what has accumulated: that is rounded once per step and not once per head
    for (int j0 = 0; j0 < a.G; j0 += kHeadsAtOnce) {
        const int nj = min(kHeadsAtOnce, a.G - j0);
        // Maximum and reciprocal sum, read once per block: read by every thread, the few words they are in held the kernel up for 5 us.
        float4 s4[kHeadsAtOnce];
#pragma unroll
        for (int j = 0; j < kHeadsAtOnce; ++j)
            if (on && j < nj) s4[j] = __ldcs(reinterpret_cast<const float4 *>(scores + (size_t)(j0 + j) * a.c.T));
        __syncthreads();
        if ((int)threadIdx.x < nj) {
            const float2 m = __ldcg(ml + j0 + threadIdx.x);
            ml_s[threadIdx.x] = make_float2(m.x, (m.y > 0.f || m.y != m.y) ? 1.0f / m.y : 0.f);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kHeadsAtOnce; ++j) {
            if (!on || j >= nj) continue;
            const float s[4] = {s4[j].x, s4[j].y, s4[j].z, s4[j].w};
            const float2 m = ml_s[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += m.y != 0.f && r + e >= begin ? ex2(s[e] - m.x) * m.y : 0.f;
        }
    }
    if (!on) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] += sum[e];
    if (r + 3 <= past) {
        *reinterpret_cast<float4 *>(a.weight_out + i) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (r + e <= past) a.weight_out[i + e] = w[e];
    }
}

template <int D, int CODE, int NT> cudaError_t launch_t(const Kv8DecodeArgs &a, cudaStream_t stream) {
    const unsigned grid = (unsigned)a.c.B * (unsigned)a.c.H * (unsigned)a.nchunk * (unsigned)a.nsplit_max;
    const bool form = a.cap_log2e > 0.f || a.slopes || a.key_begin;
    constexpr int smem = kWarps * Ring<D>::kWarpBytes;
    static_assert(smem >= kWarps * 4 * NT * (D + 16) * (int)sizeof(float), "the warps' results take the rings' room");
    auto kern = form ? flb_kv8_decode_kernel<D, CODE, NT, true> : flb_kv8_decode_kernel<D, CODE, NT, false>;
    // the shared-memory opt-in is a property of (kernel, device): set once per device
    static std::atomic<unsigned long long> opted_in[2] = {{0}, {0}};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = (dev >= 0 && dev < 64) ? (1ull << dev) : 0ull;
    if (!(opted_in[form].load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (bit) opted_in[form].fetch_or(bit, std::memory_order_release);
    }
    e = kv8_launch(kern, grid, kWarps * 32, smem, stream, a);
    if (e != cudaSuccess || !a.weight_out) return e;
    const int rows = min(a.c.T, a.nsplit_max * a.split_len), bpu = (rows + 1023) / 1024;
    return kv8_launch(flb_kv8_weights_kernel, (unsigned)a.c.B * (unsigned)a.c.H * (unsigned)bpu, 256, 0, stream, a, bpu);
}

template <int CODE> cudaError_t launch_code(const Kv8DecodeArgs &a, int d, int nt, cudaStream_t stream) {
    if (d == 256) return launch_t<256, CODE, 1>(a, stream);
    if (d == 64) return nt == 2 ? launch_t<64, CODE, 2>(a, stream) : launch_t<64, CODE, 1>(a, stream);
    return nt == 2 ? launch_t<128, CODE, 2>(a, stream) : launch_t<128, CODE, 1>(a, stream);
}

} // namespace

cudaError_t launch_kv8_decode(const Kv8DecodeArgs &a, int d, int code, int nt, cudaStream_t stream) {
    return code == kCodeI8 ? launch_code<kCodeI8>(a, d, nt, stream) : launch_code<kCodeE4M3>(a, d, nt, stream);
}

} // namespace flb
