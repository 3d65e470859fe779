// kv8_evict.cu — the cached rows that drew the least attention leave, the others close up.
//
// 1. flb_kv8_select_kernel, one CTA per K/V head: which rows stay.  A radix selection over the weights (as ordered
//    integers) finds the smallest kept weight and how many rows of exactly that weight stay (the lowest of them); one pass
//    in row order then lists the holes below m = min(n, budget) and the kept rows behind it.
// 2. flb_kv8_move_kernel, one CTA per block of rows with a hole, K and V apart: the i-th hole takes the i-th
//    kept row from behind m.  Sources lie at or behind m and targets below it, so nothing waits for anything.  The
//    block's scale grows by the rule of an append (32 values per thread, held in registers in between).
// Filling holes moves at most n - m rows and recodes only those (and a block whose scale grows); closing the gaps in row order
// would move nearly every row and round nearly every code once more at each eviction.
#include "kv8.cuh"

namespace flb {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kRowsPerThread = 4; // a thread's rows of a pass are neighbours

// weights as integers of the same order; NaN above everything
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w); // -0 equals 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ bool is_safe(const Kv8EvictArgs &a, int pos, int next) {
    return pos < a.sinks || (a.next_pos && (long long)pos >= (long long)next - a.recent);
}

// sum over the block in thread order: exclusive prefix of this thread and the total.  `ws`: one word per warp + 1.
__device__ __forceinline__ int block_scan(int v, int *ws, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
    }
    if (lane == 31) ws[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int s = ws[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, s, off);
            if (lane >= off) s += o;
        }
        ws[lane] = s;
    }
    __syncthreads();
    const int before = warp ? ws[warp - 1] : 0;
    total = ws[31];
    __syncthreads();
    return before + inc - v;
}

__global__ void __launch_bounds__(kSelThreads) flb_kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    __shared__ int hist[256];
    __shared__ int ws[32];
    __shared__ int sh_digit, sh_above, sh_safe;
    const size_t unit = blockIdx.x;
    const int b = (int)(unit / a.c.H);
    const int tid = threadIdx.x;
    int *off = a.hole_off + unit * (a.c.nblk + 1);
    int n = a.past_lens ? __ldg(a.past_lens + b) : a.start_pos;
    if (n < 0 || n > a.c.T) { // flagged; the sequence is left alone
        if (tid == 0) atomicOr(a.status, kKv8BadLen);
        for (int j = tid; j <= a.c.nblk; j += kSelThreads) off[j] = 0;
        return;
    }
    const int m = min(n, a.budget);
    if (n <= a.budget) {
        for (int j = tid; j <= a.c.nblk; j += kSelThreads) off[j] = 0;
        return;
    }
    const float *w = a.weight + unit * a.c.T;
    const int *pos = a.c.row_pos + unit * a.c.T;
    const int next = a.next_pos ? __ldg(a.next_pos + b) : 0;

    // Sources may share a block with targets, the one that row m lies in.  Its rows from m on are left as they are and the scale
    // they were coded with is kept aside, so the order in which the blocks are filled does not matter.
    if (tid < 2) a.edge_scale[unit * 2 + tid] = a.c.scale[tid][unit * a.c.nblk + (m >> a.c.block_shift)];

    // protected rows
    if (tid == 0) sh_safe = 0;
    __syncthreads();
    {
        int c = 0;
        for (int r = tid; r < n; r += kSelThreads) c += is_safe(a, pos[r], next);
        c = __reduce_add_sync(0xffffffffu, c);
        if ((tid & 31) == 0 && c) atomicAdd(&sh_safe, c);
    }
    __syncthreads();
    // More protected rows than room (positions given twice): the selection is among them.  Else they all stay and it is among the others.
    const bool among_safe = sh_safe > m;
    int want = among_safe ? m : m - sh_safe; // rows to select
    uint32_t prefix = 0, mask = 0;
    int above = 0; // rows of a larger weight than the prefix allows
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int r = tid; r < n; r += kSelThreads) {
            const uint32_t k = ordered(w[r]);
            if (is_safe(a, pos[r], next) == among_safe && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid < 32) { // the digit at which the count from above reaches `want`: lane i holds the bins 255 - 8 i and below
            int s[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += s[i] = hist[255 - 8 * tid - i];
            int inc = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, off);
                if (tid >= off) inc += v;
            }
            const unsigned reach = __ballot_sync(0xffffffffu, above + inc >= want);
            if (tid == __ffs(reach) - 1) {
                int c = above + inc - sum, d = 255 - 8 * tid;
                bool found = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    found = found || c + s[i] >= want;
                    if (!found) {
                        c += s[i];
                        --d;
                    }
                }
                sh_digit = d;
                sh_above = c;
            }
        }
        __syncthreads();
        prefix |= (uint32_t)sh_digit << shift;
        mask |= 255u << shift;
        above = sh_above;
        __syncthreads();
    }
    const uint32_t least = prefix;       // smallest kept weight; above it everything stays
    const int equals = want - above;     // so many rows of that weight stay, the lowest ones (none when want is 0)

    int seen = 0, holes = 0, kept_behind = 0;
    int *hole_list = a.holes + unit * (a.c.T / 2), *move_list = a.moves + unit * (a.c.T / 2);
    for (int base = 0; base < n; base += kSelThreads * kRowsPerThread) {
        const int r0 = base + tid * kRowsPerThread;
        uint32_t eq = 0, keep = 0; // bit i: row r0 + i
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int r = r0 + i;
            if (r >= n) continue;
            const bool safe = is_safe(a, pos[r], next);
            if (safe != among_safe) {
                if (safe) keep |= 1u << i;
                continue;
            }
            const uint32_t k = ordered(w[r]);
            if (k > least) keep |= (want > 0) ? 1u << i : 0u;
            else if (k == least) eq |= 1u << i;
        }
        int total;
        int e = seen + block_scan(__popc(eq), ws, total);
        seen += total;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i)
            if (eq >> i & 1u) {
                if (e < equals) keep |= 1u << i;
                ++e;
            }
        uint32_t hole = 0, from = 0;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int r = r0 + i;
            if (r < m) hole |= (~keep >> i & 1u) << i;
            else if (r < n) from |= (keep >> i & 1u) << i;
        }
        int hrank = holes + block_scan(__popc(hole), ws, total);
        holes += total;
        int frank = kept_behind + block_scan(__popc(from), ws, total);
        kept_behind += total;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int r = r0 + i;
            if (r <= m && (r & ((1 << a.c.block_shift) - 1)) == 0) off[r >> a.c.block_shift] = hrank;
            if (hole >> i & 1u) hole_list[hrank++] = r;
            if (from >> i & 1u) move_list[frank++] = r;
        }
    }
    // blocks from the one behind row m on: no holes
    const int first = (m + (1 << a.c.block_shift) - 1) >> a.c.block_shift;
    for (int j = first + tid; j <= a.c.nblk; j += kSelThreads) off[j] = holes;
}

constexpr int kChunks = 4; // 8-code chunks per thread

template <int D, int CODE> __global__ void __launch_bounds__(1024) flb_kv8_move_kernel(const __grid_constant__ Kv8EvictArgs a) {
    constexpr int CPR = D / 8;
    __shared__ uint32_t red[32];
    __shared__ int from_s[128]; // source of every row of the block, -1 = stays
    unsigned id = blockIdx.x;
    const int kv = (int)(id & 1u);
    id >>= 1;
    const int blk = (int)(id % (unsigned)a.c.nblk);
    const size_t unit = id / (unsigned)a.c.nblk;
    const int b = (int)(unit / a.c.H);
    const int n = a.past_lens ? __ldg(a.past_lens + b) : a.start_pos;
    if (n < 0 || n > a.c.T) return;
    const int m = min(n, a.budget);
    const int rows = 1 << a.c.block_shift, row0 = blk << a.c.block_shift;
    if (row0 >= m) return;
    const int lo = a.hole_off[unit * (a.c.nblk + 1) + blk], hi = a.hole_off[unit * (a.c.nblk + 1) + blk + 1];
    const int *hole_list = a.holes + unit * (a.c.T / 2), *move_list = a.moves + unit * (a.c.T / 2);
    const size_t urow = unit * a.c.T;
    const bool along = kv == 0 && (lo < hi || a.weight_out != a.weight || a.pos_out != a.c.row_pos);
    if (lo >= hi && !along) return;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) from_s[i] = -1;
    __syncthreads();
    for (int i = lo + (int)threadIdx.x; i < hi; i += blockDim.x) from_s[hole_list[i] - row0] = move_list[i];
    __syncthreads();
    if (along) {
        for (int i = threadIdx.x; i < rows && row0 + i < m; i += blockDim.x) {
            const int src = from_s[i] < 0 ? row0 + i : from_s[i];
            const float w = a.weight[urow + src];
            const int p = a.c.row_pos[urow + src];
            a.weight_out[urow + row0 + i] = w;
            a.pos_out[urow + row0 + i] = p;
        }
    }
    if (lo >= hi) return;

    const uint8_t *all = a.c.codes[kv] + urow * D;
    uint2 *mine = reinterpret_cast<uint2 *>(a.c.codes[kv] + (urow + row0) * D);
    const float *scales = a.c.scale[kv] + unit * a.c.nblk;
    float x[kChunks][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int ch = threadIdx.x + i * blockDim.x, src = from_s[ch / CPR];
        if (src >= 0) {
            const uint2 u = *reinterpret_cast<const uint2 *>(all + (size_t)src * D + (ch % CPR) * 8);
            const float s = (src >> a.c.block_shift) == (m >> a.c.block_shift) ? a.edge_scale[unit * 2 + kv] : scales[src >> a.c.block_shift];
            float p[4], q[4];
            kv8_decode4<CODE>(u.x, p);
            kv8_decode4<CODE>(u.y, q);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = __fmul_rn(e < 4 ? p[e & 3] : q[e & 3], s);
                amax = max(amax, kv8_abs_bits(x[i][e]));
            }
        }
    }
    amax = kv8_block_max(amax, red);
    const float old = scales[blk];
    __syncthreads(); // the old scale has been read
    const float scale = kv8_new_scale<CODE>(amax, old);
    const bool grown = old > 0.f && scale > old;
    const float ratio = grown ? __fdiv_rn(old, scale) : 1.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int ch = threadIdx.x + i * blockDim.x;
        if (from_s[ch / CPR] >= 0)
            mine[ch] = kv8_encode8<CODE>(x[i], scale);
        else if (grown && row0 + ch / CPR < m)
            mine[ch] = kv8_rescale8<CODE>(mine[ch], ratio);
    }
    if (threadIdx.x == 0) a.c.scale[kv][unit * a.c.nblk + blk] = scale;
}

__global__ void flb_kv8_lens_kernel(const __grid_constant__ Kv8EvictArgs a) {
    for (int b = threadIdx.x; b < a.c.B; b += blockDim.x) {
        const int n = a.past_lens ? a.past_lens[b] : a.start_pos;
        a.len_out[b] = (n < 0 || n > a.c.T) ? n : min(n, a.budget);
    }
}

template <int D, int CODE> cudaError_t launch_t(const Kv8EvictArgs &a, cudaStream_t stream) {
    const unsigned units = (unsigned)a.c.B * (unsigned)a.c.H;
    flb_kv8_select_kernel<<<units, kSelThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    flb_kv8_move_kernel<D, CODE><<<units * (unsigned)a.c.nblk * 2u, (unsigned)((D << a.c.block_shift) / (8 * kChunks)), 0, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    flb_kv8_lens_kernel<<<1, 256, 0, stream>>>(a); // last: len_out may be past_lens
    return cudaGetLastError();
}

} // namespace

cudaError_t launch_kv8_evict(const Kv8EvictArgs &a, int d, int code, cudaStream_t stream) {
    if (code == kCodeI8) {
        if (d == 64) return launch_t<64, kCodeI8>(a, stream);
        if (d == 256) return launch_t<256, kCodeI8>(a, stream);
        return launch_t<128, kCodeI8>(a, stream);
    }
    if (d == 64) return launch_t<64, kCodeE4M3>(a, stream);
    if (d == 256) return launch_t<256, kCodeE4M3>(a, stream);
    return launch_t<128, kCodeE4M3>(a, stream);
}

} // namespace flb
