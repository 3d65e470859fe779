// kv8_append.cu — fresh K/V rows into the 8-bit cache: dequantise, rotate (RoPE), one scale per block of rows and head.
//
// A streaming pass: a token row and head costs 2 d (e_in + 1) bytes.  Bound by instruction issue, about 100 per eight values at 2.6 a clock (8 x 32 heads of
// 0-1024 fp16 tokens to int8: 33-36 us by the lengths drawn, 3.2-3.5 TB/s, 0.50-0.54 of the copy bandwidth).  One CTA takes one block of rows of one head, K or V:
// block_len * d values, 32 per thread held in registers between the two halves of the work (largest magnitude, then
// codes), so every value is read once.  Blocks of the K/V heads of the same tokens are neighbours in the grid: together
// they read whole rows of the [B,S,Hkv,d] input.
#include "kv8.cuh"

#include <climits>
#include <type_traits>

namespace flb {

namespace {

constexpr int kChunks = 4; // 8-value chunks per thread (the call above, same lengths: 2: 40.0 us, 4: 32.0, 8: 39.0)

template <int D, int CODE, int MODE> __global__ void __launch_bounds__(1024) flb_kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a) {
    constexpr int CPR = D / 8; // chunks per row
    __shared__ uint32_t red[32];
    kv8_begin();
    const int kv = (int)(blockIdx.x & 1u), h = (int)(blockIdx.x >> 1), j = (int)blockIdx.y, b = (int)blockIdx.z;

    const int past = a.past_lens ? a.past_lens[b] : a.start_pos;
    const int n = a.new_lens ? a.new_lens[b] : a.S;
    if (past < 0 || n < 0 || n > a.S || past > min(a.c.T - n, a.max_past)) { // nothing of this sequence is touched
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, kKv8BadLen);
        return;
    }
    const int blk = (past >> a.c.block_shift) + j;
    const int row0 = blk << a.c.block_shift, row1 = row0 + (1 << a.c.block_shift);
    const int lo = max(past, row0), hi = min(past + n, row1); // new rows of this block
    if (lo >= hi) return;

    const size_t unit = (size_t)b * a.c.H + h;
    uint8_t *codes = a.c.codes[kv] + (unit * a.c.T + row0) * D;
    float *scale_p = a.c.scale[kv] + unit * a.c.nblk + blk;
    const long long pos_lo = (a.token_pos ? a.token_pos[b] : past) + (long long)(lo - past); // position of row lo: any int, and the tokens behind it further

    const int col = (int)(threadIdx.x % CPR) * 8, step = (int)(blockDim.x / CPR), r0 = row0 + (int)(threadIdx.x / CPR); // rows r0, r0 + step, ...
    // All loads first: the rows, then the table's.  What is not a new row of this block is read as the nearest that is, and not used.  FULL: every
    // row of the block is new, as in most of a prompt.
    auto work = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        auto row_of = [&](int i) { return FULL ? r0 + i * step : min(max(r0 + i * step, lo), hi - 1); };
        Kv8Raw raw[kChunks];
        float4 f0[kChunks], f1[kChunks];
        const bool turn = kv == 0 && a.freq_cis;
        const int tab1 = a.freq_rows - 1, tab_lo = (int)min(max(pos_lo, -128ll), INT_MAX - 128ll); // (a block holds 128 rows or fewer)
        if (turn && threadIdx.x == 0 && (pos_lo < 0 || pos_lo + (hi - 1 - lo) > tab1) && a.status) atomicOr(a.status, kKv8BadPos);
        const size_t tok0 = (size_t)b * a.S + (lo - past);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int row = row_of(i);
            raw[i] = kv8_raw8<MODE>(a.in[kv], tok0 + (row - lo), h * D + col);
            if (turn) {
                const float4 *f = reinterpret_cast<const float4 *>(a.freq_cis + (size_t)min(max(tab_lo + (row - lo), 0), tab1) * D + col);
                f0[i] = f[0];
                f1[i] = f[1];
            }
        }
        const float old = (FULL || row0 >= past) ? 0.f : *scale_p;
        float x[kChunks][8];
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            kv8_values8<MODE>(raw[i], a.in[kv], a.act_scale, tok0 + (row_of(i) - lo), h * D + col, x[i]);
            if (turn) kv8_rotate8(f0[i], f1[i], x[i]);
            big = kv8_abs_max8(big, x[i]); // rows read in place of others are rows of this block: the maximum is the same
        }
        const uint32_t amax = kv8_block_max(kv8_abs_bits(big), red);
        __syncthreads(); // every thread has read the old scale
        const float scale = kv8_new_scale<CODE>(amax, old);
        const bool grown = old > 0.f && scale > old;
        const float ratio = grown ? __fdiv_rn(old, scale) : 1.f, inv = __fdiv_rn(1.f, scale);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int row = r0 + i * step;
            uint2 *dst = reinterpret_cast<uint2 *>(codes) + threadIdx.x + i * blockDim.x;
            if (FULL || (row >= lo && row < hi))
                *dst = kv8_encode8<CODE>(x[i], scale, inv);
            else if (!FULL && row < past && grown)
                *dst = kv8_rescale8<CODE>(*dst, ratio);
        }
        if (threadIdx.x == 0) *scale_p = scale;
    };
    if (lo == row0 && hi == row1)
        work(std::true_type());
    else
        work(std::false_type());
    if (kv == 0 && a.c.row_pos)
        for (int r = lo + (int)threadIdx.x; r < hi; r += blockDim.x) a.c.row_pos[unit * a.c.T + r] = (int)min(pos_lo + (r - lo), (long long)INT_MAX);
}

template <int D, int CODE> cudaError_t launch_t(const Kv8AppendArgs &a, int input_mode, cudaStream_t stream) {
    const unsigned threads = (unsigned)((D << a.c.block_shift) / (8 * kChunks));
    const dim3 grid(2u * (unsigned)a.c.H, (unsigned)a.nwin, (unsigned)a.c.B);
    auto kern = input_mode == 0 ? flb_kv8_append_kernel<D, CODE, 0> : input_mode == 1 ? flb_kv8_append_kernel<D, CODE, 1> : flb_kv8_append_kernel<D, CODE, 2>;
    return kv8_launch(kern, grid, threads, 0, stream, a);
}

} // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs &a, int d, int code, int input_mode, cudaStream_t stream) {
    if (code == kCodeI8) {
        if (d == 64) return launch_t<64, kCodeI8>(a, input_mode, stream);
        if (d == 256) return launch_t<256, kCodeI8>(a, input_mode, stream);
        return launch_t<128, kCodeI8>(a, input_mode, stream);
    }
    if (d == 64) return launch_t<64, kCodeE4M3>(a, input_mode, stream);
    if (d == 256) return launch_t<256, kCodeE4M3>(a, input_mode, stream);
    return launch_t<128, kCodeE4M3>(a, input_mode, stream);
}

} // namespace flb
