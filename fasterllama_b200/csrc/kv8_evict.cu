// kv8_evict.cu — the cached rows that drew the least attention leave, the others close up.
//
// 1. flb_kv8_select_kernel, a CTA or a cluster of eight per K/V head: which rows stay.  A radix selection over the weights (as ordered
//    integers, in registers; histograms meet in distributed shared memory) finds the smallest kept weight and how many rows of
//    exactly that weight stay (the lowest of them); prefix sums in row order then list the holes below m = min(n, budget) and
//    the kept rows behind it, and weights and positions move.
// 2. flb_kv8_move_kernel, K and V apart, a CTA per four blocks of rows: the i-th hole takes the i-th
//    kept row from behind m.  Sources lie at or behind m and targets below it, so nothing waits for anything.  The
//    block's scale grows by the rule of an append (the codes are held in registers in between).
// Filling holes moves at most n - m rows and recodes only those (and a block whose scale grows); closing the gaps in row order
// would move nearly every row and round nearly every code once more at each eviction.
#include "kv8.cuh"

#include <cooperative_groups.h>

#include <climits>
#include <type_traits>

namespace flb {

namespace cg = cooperative_groups;

namespace {

constexpr int kSelThreads = 1024;
constexpr int kRanks = 8;    // CTAs of a cluster, where there is more than one
constexpr int kRegRows = 16; // rows whose keys a thread keeps in registers
// Digits of 12, 10 and 10 bits: sign, exponent and the first mantissa bits first, which leaves a percent of the rows for the other passes and spreads
// the additions of the first one over more words than a byte would.
constexpr int kBins = 4096, kBins2 = 1024;

// weights as integers of the same order; NaN above everything
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w); // -0 equals 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}


// Exclusive prefix over the block in thread order, and the total.  `ws`: a word per warp.
template <typename T> __device__ __forceinline__ T block_scan(T v, T *ws, T &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T o = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += o;
    }
    if (lane == 31) ws[warp] = inc;
    __syncthreads();
    T s = ws[lane]; // every warp adds the warps up for itself
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T o = __shfl_up_sync(0xffffffffu, s, off);
        if (lane >= off) s += o;
    }
    total = __shfl_sync(0xffffffffu, s, 31);
    const T before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
    __syncthreads(); // `ws` may be written again
    return (warp ? before : 0) + inc - v;
}

// A barrier over the cluster; a cluster of one needs no more than its own.
__device__ __forceinline__ void all_sync(cg::cluster_group &cluster, int ranks) {
    if (ranks == 1)
        __syncthreads();
    else
        cluster.sync();
}

// A cluster of CTAs (one, for short slabs) per K/V head; every thread has `per` neighbouring rows.  REGS: their keys stay in registers over
// the passes; else (beyond 16 rows a thread) they are read again.
template <bool REGS> __global__ void __launch_bounds__(kSelThreads) flb_kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    __shared__ __align__(16) int hist[kBins];                  // leading digit, then the two others
    __shared__ int hist2[2][kBins2];
    __shared__ long long ws[32];
    __shared__ int wi[32];
    __shared__ int n_safe;
    __shared__ int n_equal;
    __shared__ int found[3];                     // digit, rows above it, rows in it
    __shared__ long long n_lists; // holes, and kept rows behind m in the upper half
    kv8_begin();
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const size_t unit = blockIdx.x / (unsigned)ranks;
    const int b = (int)(unit / a.c.H);
    const int tid = threadIdx.x, lane = tid & 31;
    int *off = a.hole_off + unit * (a.c.nblk + 1);
    const float *w = a.weight + unit * a.c.T;
    const int *pos = a.c.row_pos + unit * a.c.T;
    float *w_out = a.weight_out + unit * a.c.T;
    int *p_out = a.pos_out + unit * a.c.T;
    // This thread's rows are r0 .. r0 + per - 1 of the slab; its weights and positions are on their way before the length is known.
    const int per = (((a.c.T + ranks - 1) / ranks + kSelThreads - 1) / kSelThreads + 3) & ~3;
    const int r0 = min(a.c.T, (rank * kSelThreads + tid) * per);
    float4 wv[REGS ? kRegRows / 4 : 1];
    int4 pv[REGS ? kRegRows / 4 : 1];
    if (REGS) {
#pragma unroll
        for (int v = 0; v < kRegRows / 4; ++v) {
            wv[v % (REGS ? kRegRows / 4 : 1)] = make_float4(0.f, 0.f, 0.f, 0.f);
            pv[v % (REGS ? kRegRows / 4 : 1)] = make_int4(0, 0, 0, 0);
            if (4 * v < per && r0 + 4 * v < a.c.T) { // rows come in fours: the slab's length is a multiple of 16
                wv[v % (REGS ? kRegRows / 4 : 1)] = *reinterpret_cast<const float4 *>(w + r0 + 4 * v);
                pv[v % (REGS ? kRegRows / 4 : 1)] = *reinterpret_cast<const int4 *>(pos + r0 + 4 * v);
            }
        }
    }
    // (through L1: every warp of every CTA reads these few words)
    const int n = a.past_lens ? a.past_lens[b] : a.start_pos;
    const long long first_recent = a.next_pos ? (long long)a.next_pos[b] - a.recent : INT_MAX + 1ll;
    const int recent_from = (int)min((long long)INT_MAX, max((long long)INT_MIN, first_recent));
    const bool any_recent = first_recent <= INT_MAX;
    auto is_safe = [&](int p) { return p < a.sinks || (any_recent && p >= recent_from); };
    const bool bad = n < 0 || n > a.c.T; // flagged; the sequence is left alone
    const int m = bad ? 0 : min(n, a.budget);
    if (tid == 0 && rank == 0) {
        a.seq_len[2 * b] = m; // the same from every head
        a.seq_len[2 * b + 1] = bad ? n : m;
    }
    // Rows below m into the results, where those are other buffers; the holes are written over at the end.
    if (w_out != w || p_out != pos) {
        if (REGS) {
#pragma unroll
            for (int v = 0; v < kRegRows / 4; ++v) {
                constexpr int V = REGS ? kRegRows / 4 : 1;
                const int r = r0 + 4 * v;
                if (4 * v >= per || r >= m) continue;
                if (r + 4 <= m) {
                    *reinterpret_cast<float4 *>(w_out + r) = wv[v % V];
                    *reinterpret_cast<int4 *>(p_out + r) = pv[v % V];
                } else {
                    const float x[4] = {wv[v % V].x, wv[v % V].y, wv[v % V].z, wv[v % V].w};
                    const int y[4] = {pv[v % V].x, pv[v % V].y, pv[v % V].z, pv[v % V].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (r + i < m) {
                            w_out[r + i] = x[i];
                            p_out[r + i] = y[i];
                        }
                }
            }
        } else {
            for (int r = r0; r < min(m, r0 + per); ++r) {
                w_out[r] = w[r];
                p_out[r] = pos[r];
            }
        }
    }
    if (bad || n <= a.budget) {
        for (int j = rank * kSelThreads + tid; j <= a.c.nblk; j += ranks * kSelThreads) off[j] = 0;
        return; // the whole cluster alike
    }
    // Sources may share a block with targets, the one that row m lies in.  Its rows from m on are left as they are and the scale
    // they were coded with is kept aside, so the order in which the blocks are filled does not matter.
    if (tid < 2 && rank == 0) a.edge_scale[unit * 2 + tid] = a.c.scale[tid][unit * a.c.nblk + (m >> a.c.block_shift)];

    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    for (int i = tid; i < 2 * kBins2; i += kSelThreads) hist2[0][i] = 0;
    if (tid == 0) n_safe = n_equal = 0;
    __syncthreads();

    const int r1 = max(r0, min(n, r0 + per));
    uint32_t key[REGS ? kRegRows : 1];
    uint32_t safe_bits = 0;
    int safe = 0;
    if (REGS) {
#pragma unroll
        for (int v = 0; v < kRegRows / 4; ++v) {
            constexpr int K = REGS ? kRegRows : 1, V = REGS ? kRegRows / 4 : 1;
            key[(4 * v) % K] = ordered(wv[v % V].x);
            key[(4 * v + 1) % K] = ordered(wv[v % V].y);
            key[(4 * v + 2) % K] = ordered(wv[v % V].z);
            key[(4 * v + 3) % K] = ordered(wv[v % V].w);
            const int4 p = pv[v % V];
            safe_bits |= (uint32_t)(is_safe(p.x) | is_safe(p.y) << 1 | is_safe(p.z) << 2 | is_safe(p.w) << 3) << (4 * v);
        }
        if (r1 - r0 < 32) safe_bits &= (1u << (r1 - r0)) - 1u;
        safe = __popc(safe_bits);
    } else {
        for (int r = r0; r < r1; ++r) safe += is_safe(pos[r]);
    }
    safe = __reduce_add_sync(0xffffffffu, safe);
    if (lane == 0 && safe) atomicAdd(&n_safe, safe);
    // f(row, key, protected) for each of this thread's rows
    auto each = [&](auto f) {
        if (REGS) {
#pragma unroll
            for (int i = 0; i < kRegRows; ++i)
                if (i < per && r0 + i < r1) f(r0 + i, key[i % (REGS ? kRegRows : 1)], (safe_bits >> i & 1u) != 0);
        } else {
            for (int r = r0; r < r1; ++r) f(r, ordered(w[r]), is_safe(pos[r]));
        }
    };
    // The digit at which the count from above reaches `want`: bins are summed over the cluster, BPT of them per thread from the largest down.
    auto find = [&](int *bins, auto per_thread, int want, int above) {
        constexpr int BPT = decltype(per_thread)::value;
        int c[BPT] = {}, sum = 0;
        const int top = (tid + 1) * -BPT + kSelThreads * BPT; // bins top .. top + BPT - 1
        auto add = [&](const int *p) {
            if (BPT == 4) {
                const int4 v = *reinterpret_cast<const int4 *>(p + top);
                c[0] += v.x;
                c[1 % BPT] += v.y;
                c[2 % BPT] += v.z;
                c[3 % BPT] += v.w;
            } else {
                c[0] += p[top];
            }
        };
        static_assert(BPT == 4 || BPT == 1, "one load per CTA of the cluster");
        if (ranks == 1) {
            add(bins);
        } else {
#pragma unroll
            for (int r = 0; r < kRanks; ++r) add(cluster.map_shared_rank(bins, r)); // independent loads: one latency
        }
#pragma unroll
        for (int i = 0; i < BPT; ++i) sum += c[i];
        int total;
        int at = above + block_scan(sum, wi, total);
        if (at < want && at + sum >= want) {
#pragma unroll
            for (int i = BPT - 1; i >= 0; --i) {
                if (at < want && at + c[i] >= want) {
                    found[0] = top + i;
                    found[1] = at;
                    found[2] = c[i];
                }
                at += c[i];
            }
        }
        __syncthreads();
    };
    // Protected rows all stay, and the selection is among the others; with more of them than room (positions given twice) it is among them.
    bool among_safe = false;
    each([&](int, uint32_t k, bool s) {
        if (!s) atomicAdd(&hist[k >> 20], 1);
    });
    all_sync(cluster, ranks);
    int all_safe = 0;
    for (int c = 0; c < ranks; ++c) all_safe += ranks == 1 ? n_safe : *cluster.map_shared_rank(&n_safe, c);
    int want = m - all_safe; // rows to select
    if (want < 0) {
        among_safe = true;
        want = m;
        all_sync(cluster, ranks); // nobody reads the histogram of the others any more
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        each([&](int, uint32_t k, bool s) {
            if (s) atomicAdd(&hist[k >> 20], 1);
        });
        all_sync(cluster, ranks);
    }
    uint32_t least = 0xffffffffu; // smallest kept weight; above it everything stays,
    int equals = 0, level = 0;    // and of it so many rows, of so many
    if (want > 0) {
        find(hist, std::integral_constant<int, kBins / kSelThreads>(), want, 0);
        uint32_t prefix = (uint32_t)found[0] << 20;
        int above = found[1];
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            const int shift = 10 - 10 * pass;
            each([&](int, uint32_t k, bool s) {
                if (s == among_safe && ((k ^ prefix) >> (shift + 10)) == 0) atomicAdd(&hist2[pass][(k >> shift) & (kBins2 - 1)], 1);
            });
            all_sync(cluster, ranks);
            find(hist2[pass], std::integral_constant<int, kBins2 / kSelThreads>(), want, above);
            prefix |= (uint32_t)found[0] << shift;
            above = found[1];
        }
        least = prefix;
        equals = want - above;
        level = found[2];
    }

    // rows of that weight in front of this thread, where not all of them stay: the lowest do
    int e = 0;
    if (equals < level) {
        int eq = 0;
        each([&](int, uint32_t k, bool s) { eq += s == among_safe && k == least; });
        int total;
        e = block_scan(eq, wi, total);
        if (tid == 0) n_equal = total;
        all_sync(cluster, ranks);
        for (int c = 0; c < rank; ++c) e += *cluster.map_shared_rank(&n_equal, c);
    }
    // holes and sources in front of this thread
    int holes = 0, behind = 0;
    const int e0 = e;
    uint32_t stay_bits = 0; // REGS: what the first look found
    auto kept = [&](uint32_t k, bool s) { // in row order
        if (s != among_safe) return s;
        if (k == least) return e++ < equals;
        return k > least && want > 0;
    };
    each([&](int r, uint32_t k, bool s) {
        const bool stay = kept(k, s);
        if (REGS) stay_bits |= (uint32_t)stay << (r - r0);
        holes += r < m && !stay;
        behind += r >= m && stay;
    });
    long long total;
    const long long before = block_scan((long long)holes | ((long long)behind << 32), ws, total);
    if (tid == 0) n_lists = total;
    all_sync(cluster, ranks);
    int hr = (int)(before & 0xffffffff), br = (int)(before >> 32), all_holes = 0;
    for (int c = 0; c < ranks; ++c) {
        const long long t = ranks == 1 ? n_lists : *cluster.map_shared_rank(&n_lists, c);
        if (c < rank) {
            hr += (int)(t & 0xffffffff);
            br += (int)(t >> 32);
        }
        all_holes += (int)(t & 0xffffffff);
    }
    e = e0;
    int *hole_list = a.holes + unit * (a.c.T / 2), *move_list = a.moves + unit * (a.c.T / 2);
    const int in_block = (1 << a.c.block_shift) - 1;
    each([&](int r, uint32_t k, bool s) {
        const bool stay = REGS ? (stay_bits >> (r - r0) & 1u) != 0 : kept(k, s);
        if (r <= m && (r & in_block) == 0) off[r >> a.c.block_shift] = hr;
        if (r < m && !stay) hole_list[hr++] = r;
        if (r >= m && stay) move_list[br++] = r;
    });
    // blocks from the one behind row m on: no holes
    for (int j = ((m + in_block) >> a.c.block_shift) + rank * kSelThreads + tid; j <= a.c.nblk; j += ranks * kSelThreads) off[j] = all_holes;
    all_sync(cluster, ranks); // the lists are whole; nobody's shared memory is read any more
    // weights and positions of the holes
    for (int i = rank * kSelThreads + tid; i < all_holes; i += ranks * kSelThreads) {
        const int to = __ldcg(hole_list + i), from = __ldcg(move_list + i);
        w_out[to] = w[from];
        p_out[to] = pos[from];
    }
}

constexpr int kChunks = 4; // 8-code chunks per thread

// Blocks that a CTA looks after, one after the other.  Measured (us, whole eviction): 16 x 8 heads of 2000-4350 rows, where most blocks have no hole and a CTA only
// looks and leaves, 1: 47.0, 2: 35.0, 3: 32.8, 4: 32.1, 11: 41.3; 8 heads of 65536 rows cut to a quarter 65.1, 61.7, 61.7, 60.4, -.
constexpr int kGroup = 4;

template <int D, int CODE> __global__ void __launch_bounds__(1024) flb_kv8_move_kernel(const __grid_constant__ Kv8EvictArgs a, int groups) {
    constexpr int CPR = D / 8;
    __shared__ uint32_t red[32];
    __shared__ int from_s[kGroup * 128]; // source of every row of the blocks, -1 = stays
    kv8_begin();
    if (blockIdx.x == 0) { // len_out may be past_lens: nobody reads that any more
        int bad = 0;
        for (int b = threadIdx.x; b < a.c.B; b += blockDim.x) {
            const int n = __ldcg(a.seq_len + 2 * b + 1);
            a.len_out[b] = n;
            bad |= n < 0 || n > a.c.T;
        }
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0) *a.status = bad ? kKv8BadLen : 0u;
    }
    unsigned id = blockIdx.x;
    const int kv = (int)(id & 1u);
    id >>= 1;
    const int blk0 = (int)(id % (unsigned)groups) * kGroup;
    const size_t unit = id / (unsigned)groups;
    const int *off = a.hole_off + unit * (a.c.nblk + 1);
    const int nb = min(kGroup, a.c.nblk - blk0);
    const int lo = __ldcg(off + blk0), hi = __ldcg(off + blk0 + nb);
    if (lo >= hi) return; // no hole in any of them
    const int m = __ldcg(a.seq_len + 2 * (int)(unit / a.c.H));
    const int rows = 1 << a.c.block_shift, edge = m >> a.c.block_shift, row0 = blk0 << a.c.block_shift;
    const int *hole_list = a.holes + unit * (a.c.T / 2), *move_list = a.moves + unit * (a.c.T / 2);
    const uint8_t *all = a.c.codes[kv] + unit * a.c.T * D;
    float *scales = a.c.scale[kv] + unit * a.c.nblk;
    for (int i = threadIdx.x; i < nb * rows; i += blockDim.x) from_s[i] = -1;
    __syncthreads();
    for (int i = lo + (int)threadIdx.x; i < hi; i += blockDim.x) from_s[__ldcg(hole_list + i) - row0] = __ldcg(move_list + i);
    __syncthreads();
    uint2 next_u[kChunks];
    float next_s[kChunks], next_old = 0.f;
    auto fetch = [&](int j) { // the rows that come into block j of the group, and the scales they bring
        next_old = scales[blk0 + j];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int ch = threadIdx.x + i * blockDim.x, src = from_s[j * rows + ch / CPR];
            if (src < 0) continue;
            next_u[i] = *reinterpret_cast<const uint2 *>(all + (size_t)src * D + (ch % CPR) * 8);
            next_s[i] = (src >> a.c.block_shift) == edge ? __ldcg(a.edge_scale + unit * 2 + kv) : scales[src >> a.c.block_shift];
        }
    };
    fetch(0);
    for (int j = 0; j < nb; ++j) {
        uint2 u[kChunks];
        float s[kChunks];
        const float old = next_old;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            u[i] = next_u[i];
            s[i] = next_s[i];
        }
        if (j + 1 < nb) fetch(j + 1); // its scale is read before anybody can get to writing it, its sources are written by nobody
        const int *from = from_s + j * rows;
        const int first = row0 + j * rows;
        uint2 *mine = reinterpret_cast<uint2 *>(a.c.codes[kv] + (unit * a.c.T + first) * D);
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (from[(threadIdx.x + i * blockDim.x) / CPR] < 0) continue;
            float x[8], big = 0.f;
            kv8_decode8<CODE>(u[i], x);
            if (fabsf(s[i]) <= 3.402823466e38f) { // rounding keeps the order: the largest product is that of the largest code
#pragma unroll
                for (int e = 0; e < 8; e += 2) big = max3(big, fabsf(x[e]), fabsf(x[e + 1]));
                amax = max(amax, kv8_abs_bits(__fmul_rn(big, s[i])));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = max(amax, kv8_abs_bits(__fmul_rn(x[e], s[i])));
            }
        }
        if (j) __syncthreads(); // `red` has been read
        amax = kv8_block_max(amax, red);
        const float scale = kv8_new_scale<CODE>(amax, old);
        const bool grown = old > 0.f && scale > old;
        const float ratio = grown ? __fdiv_rn(old, scale) : 1.f, inv = __fdiv_rn(1.f, scale);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int ch = threadIdx.x + i * blockDim.x;
            if (from[ch / CPR] >= 0) {
                float x[8];
                kv8_decode8<CODE>(u[i], x);
                kv8_scale8(x, s[i]);
                mine[ch] = kv8_encode8<CODE>(x, scale, inv);
            } else if (grown && first + ch / CPR < m) {
                mine[ch] = kv8_rescale8<CODE>(mine[ch], ratio);
            }
        }
        // a block behind m, whose scale others read, never gets here with a new one
        if (threadIdx.x == 0 && __float_as_uint(scale) != __float_as_uint(old)) scales[blk0 + j] = scale;
    }
}

template <int D, int CODE> cudaError_t launch_t(const Kv8EvictArgs &a, cudaStream_t stream) {
    const unsigned units = (unsigned)a.c.B * (unsigned)a.c.H;
    // One CTA per head up to 8192 rows, eight beyond (a portable cluster); up to 16 rows per thread keys stay in registers.
    const int ranks = a.c.T <= 8192 ? 1 : kRanks;
    const bool regs = (long long)a.c.T <= (long long)ranks * kSelThreads * kRegRows;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units * (unsigned)ranks);
    cfg.blockDim = dim3(kSelThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, regs ? flb_kv8_select_kernel<true> : flb_kv8_select_kernel<false>, a);
    if (e != cudaSuccess) return e;
    const int kept_blocks = (min(a.c.T, a.budget) + (1 << a.c.block_shift) - 1) >> a.c.block_shift;
    const int groups = (kept_blocks + kGroup - 1) / kGroup;
    return kv8_launch(flb_kv8_move_kernel<D, CODE>, units * (unsigned)groups * 2u, (unsigned)((D << a.c.block_shift) / (8 * kChunks)), 0, stream, a, groups);
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
