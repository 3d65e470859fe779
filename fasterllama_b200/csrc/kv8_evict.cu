// kv8_evict.cu — the cached rows that drew the least attention leave, the others close up.
//
// 1. flb_kv8_select_kernel, a CTA or a cluster of eight per K/V head: which rows stay.  A radix selection over the weights (as ordered
//    integers, in registers; histograms meet in distributed shared memory) finds the smallest kept weight and how many rows of
//    exactly that weight stay (the lowest of them); one prefix sum in row order then lists the holes below m = min(n, budget) and
//    the kept rows behind it, and weights and positions move.  Bound by the chain of its steps: 10 us for slabs of 4352 rows on one CTA
//    each, 18 us for 65536 rows on eight.
// 2. flb_kv8_move_kernel, K and V apart, a CTA per four blocks of rows: the i-th hole takes the i-th
//    kept row from behind m.  Sources lie at or behind m and targets below it, so nothing waits for anything.  The
//    block's scale grows by the rule of an append (the codes are held in registers in between).  Bound by instruction issue where
//    most rows of a block are filled (about 120 per eight codes): 28 us for 98304 rows of 128
//    codes coming in, K and V.
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
// Digits of 12, 10 and 10 bits: sign, exponent and the first mantissa bits first, which leaves some percent of the rows for the other passes and
// spreads the additions of the first one over more words than a byte would.
constexpr int kBins = 4096, kBins2 = 1024;

// rows of a slab that a thread looks after, in fours
__host__ __device__ inline int rows_per_thread(int T, int ranks) { return (((T + ranks - 1) / ranks + kSelThreads - 1) / kSelThreads + 3) & ~3; }

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

// A cluster of CTAs (one, for short slabs) per K/V head; every thread has `per` neighbouring rows.  ROWS: so many of them at most, whose keys stay in
// registers over the passes; 0: any number, read again.  With 32 warps on an SM every instruction per row is eight clocks, so code
// for 16 rows does not serve where 8 do.
template <int ROWS> __global__ void __launch_bounds__(kSelThreads) flb_kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    constexpr bool REGS = ROWS > 0;
    constexpr int K = REGS ? ROWS : 4, V = K / 4;
    // Counts of the leading digit, then the candidates (the cluster's, this CTA's); counts of the two other digits; at the end both are the lists' room.
    constexpr int kPool = kBins + 2 * kBins2, kListWords = ROWS * kSelThreads / 2;
    __shared__ __align__(16) int pool[kPool > kListWords ? kPool : kListWords];
    int *const hist = pool, *const hist2 = pool + kBins;
    __shared__ long long ws[32];
    __shared__ int wi[32];
    __shared__ int n_safe, n_cand, slice_total, kept_below; // kept_below: kept rows in front of row m
    __shared__ uint32_t found[3];                 // digit or key, rows above it, rows of it
    __shared__ long long n_kept;                  // of this CTA: rows that stay for certain; rows of the smallest kept weight in the upper half
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
    const int per = rows_per_thread(a.c.T, ranks);
    const int r0 = min(a.c.T, (rank * kSelThreads + tid) * per);
    float4 wv[V];
    int4 pv[V];
    if (REGS) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            wv[v] = make_float4(0.f, 0.f, 0.f, 0.f);
            pv[v] = make_int4(0, 0, 0, 0);
            if (4 * v < per && r0 + 4 * v < a.c.T) { // rows come in fours: the slab's length is a multiple of 16
                wv[v] = *reinterpret_cast<const float4 *>(w + r0 + 4 * v);
                pv[v] = *reinterpret_cast<const int4 *>(pos + r0 + 4 * v);
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
    for (int i = tid; i < kPool / 4; i += kSelThreads) reinterpret_cast<int4 *>(pool)[i] = make_int4(0, 0, 0, 0);
    if (tid == 0) n_safe = n_cand = 0;
    // Rows below m into the results, where those are other buffers; the holes are written over at the end.
    if (w_out != w || p_out != pos) {
        if (REGS) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int r = r0 + 4 * v;
                if (4 * v >= per || r >= m) continue;
                if (r + 4 <= m) {
                    *reinterpret_cast<float4 *>(w_out + r) = wv[v];
                    *reinterpret_cast<int4 *>(p_out + r) = pv[v];
                } else {
                    const float x[4] = {wv[v].x, wv[v].y, wv[v].z, wv[v].w};
                    const int y[4] = {pv[v].x, pv[v].y, pv[v].z, pv[v].w};
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
    __syncthreads();

    const int r1 = max(r0, min(n, r0 + per));
    const uint32_t all_bits = r1 - r0 < 32 ? (1u << (r1 - r0)) - 1u : ~0u; // (REGS) this thread's cached rows
    uint32_t key[K];
    uint32_t safe_bits = 0;
    int safe = 0;
    if (REGS) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            key[4 * v] = ordered(wv[v].x);
            key[4 * v + 1] = ordered(wv[v].y);
            key[4 * v + 2] = ordered(wv[v].z);
            key[4 * v + 3] = ordered(wv[v].w);
            const int4 p = pv[v];
            safe_bits |= (uint32_t)(is_safe(p.x) | is_safe(p.y) << 1 | is_safe(p.z) << 2 | is_safe(p.w) << 3) << (4 * v);
        }
        safe_bits &= all_bits;
        safe = __popc(safe_bits);
    } else {
        for (int r = r0; r < r1; ++r) safe += is_safe(pos[r]);
    }
    safe = __reduce_add_sync(0xffffffffu, safe);
    if (lane == 0 && safe) atomicAdd(&n_safe, safe);
    // f(key) for each of this thread's rows that are protected, or that are not
    auto each = [&](bool protected_, auto f) {
        if (REGS) {
            const uint32_t bits = (protected_ ? safe_bits : ~safe_bits) & all_bits;
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (bits >> i & 1u) f(key[i]);
        } else {
            for (int r = r0; r < r1; ++r)
                if (is_safe(pos[r]) == protected_) f(ordered(w[r]));
        }
    };
    auto to_all = [&](auto *p, auto value) { // into the same word of every CTA
        for (int c = 0; c < ranks; ++c) *(ranks == 1 ? p : cluster.map_shared_rank(p, c)) = value;
    };
    // The leading digit at which the count from above reaches `want`.  Bins are summed over the cluster, by each CTA an eighth of them; four bins per thread
    // in a CTA alone.
    auto find = [&](int want) {
        if (ranks == 1) {
            const int top = kBins - 4 * (tid + 1);
            static_assert(kBins == 4 * kSelThreads, "four bins per thread");
            const int4 v = *reinterpret_cast<const int4 *>(hist + top);
            const int c[4] = {v.x, v.y, v.z, v.w};
            int total, at = block_scan(v.x + v.y + v.z + v.w, wi, total);
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                if (at < want && at + c[i] >= want) {
                    found[0] = top + i;
                    found[1] = at;
                    found[2] = c[i];
                }
                at += c[i];
            }
        } else {
            constexpr int kSlice = kBins / kRanks;
            static_assert(kSlice <= kSelThreads, "one bin per thread");
            const int bin = kBins - rank * kSlice - 1 - tid;
            int sum = 0;
            if (tid < kSlice) {
#pragma unroll
                for (int c = 0; c < kRanks; ++c) sum += *cluster.map_shared_rank(hist + bin, c); // independent loads: one latency
            }
            int total, at = block_scan(sum, wi, total);
            if (tid == 0) slice_total = total;
            cluster.sync();
#pragma unroll
            for (int c = 0; c < kRanks; ++c) at += c < rank ? *cluster.map_shared_rank(&slice_total, c) : 0;
            if (tid < kSlice && at < want && at + sum >= want) {
                to_all(found, (uint32_t)bin);
                to_all(found + 1, (uint32_t)at);
                to_all(found + 2, (uint32_t)sum);
            }
        }
        all_sync(cluster, ranks);
    };
    // The same for one of the digits of 10 bits, a bin per thread; `across`: the bins of all CTAs are summed, else these are counts of everything.
    auto find2 = [&](const int *bins, bool across, int want, int above) {
        static_assert(kBins2 == kSelThreads, "one bin per thread");
        const int bin = kBins2 - 1 - tid;
        int sum = 0, total;
        if (across && ranks > 1) {
#pragma unroll
            for (int c = 0; c < kRanks; ++c) sum += *cluster.map_shared_rank(bins + bin, c);
        } else {
            sum = bins[bin];
        }
        const int at = above + block_scan(sum, wi, total);
        if (at < want && at + sum >= want) {
            found[0] = bin;
            found[1] = at;
        }
        __syncthreads();
    };
    // Protected rows all stay, and the selection is among the others; with more of them than room (positions given twice) it is among them.
    bool among_safe = false;
    each(false, [&](uint32_t k) { atomicAdd(&hist[k >> 20], 1); });
    all_sync(cluster, ranks);
    int all_safe = 0;
    for (int c = 0; c < ranks; ++c) all_safe += ranks == 1 ? n_safe : *cluster.map_shared_rank(&n_safe, c);
    int want = m - all_safe; // rows to select
    if (want < 0) {
        among_safe = true;
        want = m;
        all_sync(cluster, ranks);
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        each(true, [&](uint32_t k) { atomicAdd(&hist[k >> 20], 1); });
        all_sync(cluster, ranks);
    }
    uint32_t least = 0xffffffffu; // smallest kept weight; above it everything stays,
    int equals = 0;               // and of it so many rows, the lowest
    if (want > 0) {
        find(want);
        uint32_t prefix = found[0] << 20;
        int above = (int)found[1];
        const int count = (int)found[2];
        static_assert(2 * kSelThreads <= kBins, "the candidates take the leading digit's room");
        const bool few = count <= kSelThreads;
        uint32_t cand = 0;
        if (few) {
            // So few rows share the leading digit with the one looked for (some percent of a slab, unless weights are equal) that each becomes a
            // thread's, in every CTA, and the other digits need no look at the rows.
            int *const all = hist, *const mine = ranks == 1 ? hist : hist + kSelThreads;
            each(among_safe, [&](uint32_t k) {
                if (((k ^ prefix) >> 20) == 0) mine[atomicAdd(&n_cand, 1)] = (int)k;
            });
            all_sync(cluster, ranks);
            if (ranks > 1) {
                int nc[kRanks], i = tid, from = kRanks;
#pragma unroll
                for (int c = 0; c < kRanks; ++c) nc[c] = *cluster.map_shared_rank(&n_cand, c);
#pragma unroll
                for (int c = 0; c < kRanks; ++c) {
                    if (from == kRanks && i < nc[c]) from = c;
                    if (from == kRanks) i -= nc[c];
                }
                if (from < kRanks) cand = (uint32_t)*cluster.map_shared_rank(mine + i, from);
            } else if (tid < count) {
                cand = (uint32_t)all[tid];
            }
        }
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            const int shift = 10 - 10 * pass;
            int *const bins = hist2 + pass * kBins2;
            auto add = [&](uint32_t k) {
                if (((k ^ prefix) >> (shift + 10)) == 0) atomicAdd(bins + ((k >> shift) & (kBins2 - 1)), 1);
            };
            if (few) {
                if (tid < count) add(cand);
                __syncthreads();
            } else {
                each(among_safe, add);
                all_sync(cluster, ranks);
            }
            find2(bins, !few, want, above);
            prefix |= found[0] << shift;
            above = (int)found[1];
        }
        least = prefix;
        equals = want - above;
    }

    // Kept rows in front of this thread: those that stay for certain (protected or heavier; or, among the protected, heavier), and the first `equals` of the
    // smallest kept weight.  Rows below m in front of r less those are the holes in front of r; kept rows behind m are counted from the last, the m-th, back.
    uint32_t sure_bits = 0, equal_bits = 0;
    int sure = 0, equal = 0;
    auto is_sure = [&](uint32_t k, bool s) { return s == among_safe ? k > least : s; };
    if (REGS) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool s = (safe_bits >> i & 1u) != 0;
            sure_bits |= (uint32_t)is_sure(key[i], s) << i;
            equal_bits |= (uint32_t)(s == among_safe && key[i] == least) << i;
        }
        sure_bits &= all_bits;
        equal_bits &= all_bits;
        sure = __popc(sure_bits);
        equal = __popc(equal_bits);
    } else {
        for (int r = r0; r < r1; ++r) {
            const uint32_t k = ordered(w[r]);
            const bool s = is_safe(pos[r]);
            sure += is_sure(k, s);
            equal += s == among_safe && k == least;
        }
    }
    long long total, first = 0; // in this CTA, and in front of it
    long long before = block_scan((long long)sure | ((long long)equal << 32), ws, total);
    if (ranks > 1) {
        if (tid == 0) n_kept = total;
        cluster.sync();
#pragma unroll
        for (int c = 0; c < kRanks; ++c) first += c < rank ? *cluster.map_shared_rank(&n_kept, c) : 0ll;
        before += first;
    }
    auto kept_of = [&](long long x) { return (int)(x & 0xffffffff) + min((int)(x >> 32), equals); };
    const int room = a.c.T / 2;
    int *hole_list = a.holes + unit * room, *move_list = a.moves + unit * room;
    const int in_block = (1 << a.c.block_shift) - 1;
    int e = (int)(before >> 32), kept = kept_of(before); // in front of the row
    // The lists are gathered in shared memory, from where they leave in order (not straight from the threads, 4 bytes
    // here and there): rows of this CTA's stretch, holes from the front, sources up to the end.
    uint16_t *const list = reinterpret_cast<uint16_t *>(pool);
    constexpr int kList = ROWS * kSelThreads;
    const int c0 = rank * kSelThreads * per, c1 = min(n, c0 + kSelThreads * per); // the stretch
    const int kept0 = kept_of(first), kept1 = kept_of(first + total);             // in front of it, and up to its end
    if (REGS) {
        uint32_t stay = sure_bits; // and the lowest of the equal ones, as many as still have room
        if (e + equal <= equals) {
            stay |= equal_bits;
        } else {
            for (uint32_t eb = equal_bits; eb && e < equals; eb &= eb - 1, ++e) stay |= eb & (0u - eb);
        }
        auto in_front = [&](int r) { return kept + __popc(stay & ((1u << (r - r0)) - 1u)); };
        const int rb = (r0 + in_block) & ~in_block; // a block that starts among these rows, of which there is one at most
        static_assert(ROWS <= 16, "blocks have 16 rows or more");
        if (rb < r1 && rb <= m) off[rb >> a.c.block_shift] = rb - in_front(rb);
        if (r0 <= m && m < r1) to_all(&kept_below, in_front(m));
        const uint32_t low = m <= r0 ? 0u : m - r0 < 32 ? (1u << (m - r0)) - 1u : ~0u; // rows below m
        const uint32_t hole_bits = ~stay & all_bits & low, source_bits = stay & ~low;
        uint16_t *h = list + ((r0 - kept) - (c0 - kept0)), *f = list + kList - (kept1 - kept - __popc(stay & low));
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (hole_bits >> i & 1u) *h++ = (uint16_t)(r0 + i - c0);
            if (source_bits >> i & 1u) *f++ = (uint16_t)(r0 + i - c0);
        }
        __syncthreads();
        if (c0 < c1) {
            const bool holds_m = c0 <= m && m < c1;
            const int below = max(0, min(m, c1) - c0); // rows of the stretch below m, and how many of those are kept
            const int kept_there = c0 >= m ? 0 : (holds_m ? kept_below : kept1) - kept0;
            const int nh = below - kept_there, ns = kept1 - kept0 - kept_there;
            for (int i = tid; i < nh; i += kSelThreads) hole_list[c0 - kept0 + i] = c0 + list[i];
            for (int i = tid; i < ns; i += kSelThreads) move_list[room - m + kept1 - ns + i] = c0 + list[kList - ns + i];
        }
    } else {
        for (int r = r0; r < r1; ++r) {
            const uint32_t k = ordered(w[r]);
            const bool s = is_safe(pos[r]), level = s == among_safe && k == least, stay = is_sure(k, s) || (level && e < equals);
            if (r <= m && (r & in_block) == 0) off[r >> a.c.block_shift] = r - kept;
            if (r == m) to_all(&kept_below, kept);
            if (r < m && !stay) hole_list[r - kept] = r;
            if (r >= m && stay) move_list[room - m + kept] = r;
            e += level;
            kept += stay;
        }
    }
    all_sync(cluster, ranks); // the lists are whole; nobody's shared memory is read or written by others any more
    const int all_holes = m - kept_below;
    // blocks from the one behind row m on: no holes
    for (int j = ((m + in_block) >> a.c.block_shift) + rank * kSelThreads + tid; j <= a.c.nblk; j += ranks * kSelThreads) off[j] = all_holes;
    // weights and positions of the holes
    for (int i = rank * kSelThreads + tid; i < all_holes; i += ranks * kSelThreads) {
        const bool own = REGS && ranks == 1;
        const int to = own ? list[i] : __ldcg(hole_list + i), from = own ? list[kList - all_holes + i] : __ldcg(move_list + room - all_holes + i);
        w_out[to] = w[from];
        p_out[to] = pos[from];
    }
}

constexpr int kChunks = 4; // 8-code chunks per thread

// Blocks that a CTA looks after.  Measured (us, whole eviction): 16 x 8 heads of 2000-4350 rows, where most blocks have few holes or none,
// 2: 26.5, 3: 22.9, 4: 21.1, 6: 20.3, 8: 21.7; 8 heads of 65536 rows cut to a quarter 50.8, 50.1, 48.7, 52.8, 50.8.
constexpr int kGroup = 4;

template <int D, int CODE> __global__ void __launch_bounds__(1024) flb_kv8_move_kernel(const __grid_constant__ Kv8EvictArgs a, int groups) {
    constexpr int CPR = D / 8;
    __shared__ uint32_t red[2][32];
    __shared__ int from_s[kGroup * 128], off_s[kGroup + 1]; // the entries of the lists that are these blocks'
    __shared__ uint16_t to_s[kGroup * 128], held_s[kGroup * 128]; // rows of the group: that are filled, that stay
    __shared__ uint32_t hole_mask[kGroup * 4];
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
    const int *hole_list = a.holes + unit * (a.c.T / 2), *move_list = a.moves + (unit + 1) * (a.c.T / 2) - __ldcg(off + a.c.nblk); // sources end with their room
    const uint8_t *all = a.c.codes[kv] + unit * a.c.T * D;
    float *scales = a.c.scale[kv] + unit * a.c.nblk;
    auto scale_of = [&](int src) { return (src >> a.c.block_shift) == edge ? __ldcg(a.edge_scale + unit * 2 + kv) : scales[src >> a.c.block_shift]; };
    if ((hi - lo) * CPR <= kChunks * (int)blockDim.x) {
        // Few holes: a thread per chunk that comes in, all blocks at once.  (Block after block the threads mostly find that a row stays.)
        __shared__ uint32_t top_s[kGroup];
        __shared__ float old_s[kGroup];
        if ((int)threadIdx.x < kGroup) {
            top_s[threadIdx.x] = 0u;
            old_s[threadIdx.x] = (int)threadIdx.x < nb ? scales[blk0 + threadIdx.x] : 0.f;
        }
        uint2 u[kChunks];
        float s[kChunks];
        int to[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int id = (int)threadIdx.x + i * (int)blockDim.x, h = lo + id / CPR;
            to[i] = -1;
            if (h < hi) {
                const int src = __ldcg(move_list + h);
                to[i] = __ldcg(hole_list + h);
                u[i] = *reinterpret_cast<const uint2 *>(all + (size_t)src * D + (id % CPR) * 8);
                s[i] = scale_of(src);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (lo + (int)(threadIdx.x + i * blockDim.x) / CPR >= hi) break; // for whole rows of chunks alike
            float x[8];
            uint32_t amax = 0;
            kv8_decode8<CODE>(u[i], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max(amax, kv8_abs_bits(__fmul_rn(x[e], s[i])));
            atomicMax(top_s + ((to[i] - row0) >> a.c.block_shift), amax);
        }
        __syncthreads();
        bool any = false;
        for (int j = 0; j < nb; ++j) {
            const float old = old_s[j], scale = kv8_new_scale<CODE>(top_s[j], old);
            if (!(old > 0.f && scale > old)) continue;
            any = true; // the codes that the block held follow; those of the holes are written over below
            uint2 *mine = reinterpret_cast<uint2 *>(a.c.codes[kv] + (unit * a.c.T + row0 + j * rows) * D);
            const float ratio = __fdiv_rn(old, scale);
            for (int ch = threadIdx.x; ch < min(rows, m - row0 - j * rows) * CPR; ch += blockDim.x) mine[ch] = kv8_rescale8<CODE>(mine[ch], ratio);
        }
        if (any) __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (to[i] < 0) break;
            const int j = (to[i] - row0) >> a.c.block_shift;
            const float scale = kv8_new_scale<CODE>(top_s[j], old_s[j]);
            float x[8];
            kv8_decode8<CODE>(u[i], x);
            kv8_scale8(x, s[i]);
            reinterpret_cast<uint2 *>(a.c.codes[kv] + (unit * a.c.T + to[i]) * D)[(threadIdx.x + i * blockDim.x) % CPR] = kv8_encode8<CODE>(x, scale, __fdiv_rn(1.f, scale));
        }
        if ((int)threadIdx.x < nb) {
            const float old = old_s[threadIdx.x], scale = kv8_new_scale<CODE>(top_s[threadIdx.x], old);
            if (__float_as_uint(scale) != __float_as_uint(old)) scales[blk0 + threadIdx.x] = scale;
        }
        return;
    }
    // Block after block, what comes in from consecutive entries of the lists and what stays from a list of its own: a warp that held rows of both kinds
    // went both ways at every chunk (whole eviction of 8 heads of 65536 rows to a quarter 51.0 us instead of 48.7).
    for (int i = threadIdx.x; i < kGroup * 4; i += blockDim.x) hole_mask[i] = 0u;
    if ((int)threadIdx.x <= nb) off_s[threadIdx.x] = __ldcg(off + blk0 + threadIdx.x) - lo;
    __syncthreads();
    for (int i = threadIdx.x; i < hi - lo; i += blockDim.x) {
        const int to = __ldcg(hole_list + lo + i) - row0, r = to & (rows - 1);
        from_s[i] = __ldcg(move_list + lo + i);
        to_s[i] = (uint16_t)to;
        atomicOr(hole_mask + (to >> a.c.block_shift) * 4 + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nb * rows; i += blockDim.x) { // rows that stay, in order
        const int j = i >> a.c.block_shift, r = i & (rows - 1), word = r >> 5;
        const uint32_t *mask = hole_mask + j * 4;
        if (row0 + i >= m || (mask[word] >> (r & 31) & 1u)) continue;
        int before = __popc(~mask[word] & ((1u << (r & 31)) - 1u));
        for (int q = 0; q < word; ++q) before += __popc(~mask[q]);
        held_s[(j << a.c.block_shift) + before] = (uint16_t)i;
    }
    __syncthreads();
    int turn = 0;
    uint2 next_u[kChunks];
    float next_s[kChunks], next_old = 0.f;
    auto fetch = [&](int j) { // the rows that come into block j of the group, and the scales they bring
        next_old = scales[blk0 + j];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int ch = threadIdx.x + i * blockDim.x, h = off_s[j] + ch / CPR;
            if (h >= off_s[j + 1]) break;
            const int src = from_s[h];
            next_u[i] = *reinterpret_cast<const uint2 *>(all + (size_t)src * D + (ch % CPR) * 8);
            next_s[i] = scale_of(src);
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
        const int coming = (off_s[j + 1] - off_s[j]) * CPR;
        if (coming == 0) continue; // for the whole block alike
        uint2 *const codes = reinterpret_cast<uint2 *>(a.c.codes[kv] + (unit * a.c.T + row0) * D);
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if ((int)(threadIdx.x + i * blockDim.x) >= coming) break;
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
        amax = kv8_block_max(amax, red[turn++ & 1]); // (the other one may still be read)
        const float scale = kv8_new_scale<CODE>(amax, old);
        const bool grown = old > 0.f && scale > old;
        const float inv = __fdiv_rn(1.f, scale);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int ch = threadIdx.x + i * blockDim.x;
            if (ch >= coming) break;
            float x[8];
            kv8_decode8<CODE>(u[i], x);
            kv8_scale8(x, s[i]);
            codes[to_s[off_s[j] + ch / CPR] * CPR + ch % CPR] = kv8_encode8<CODE>(x, scale, inv);
        }
        if (grown) { // the codes that the block holds follow its scale
            const float ratio = __fdiv_rn(old, scale);
            const int staying = (min(rows, m - row0 - j * rows) - (off_s[j + 1] - off_s[j])) * CPR;
            for (int ch = threadIdx.x; ch < staying; ch += blockDim.x) {
                uint2 *mine = codes + held_s[j * rows + ch / CPR] * CPR + ch % CPR;
                *mine = kv8_rescale8<CODE>(*mine, ratio);
            }
        }
        // a block behind m, whose scale others read, never gets here with a new one
        if (threadIdx.x == 0 && __float_as_uint(scale) != __float_as_uint(old)) scales[blk0 + j] = scale;
    }
}

template <int D, int CODE> cudaError_t launch_t(const Kv8EvictArgs &a, cudaStream_t stream) {
    const unsigned units = (unsigned)a.c.B * (unsigned)a.c.H;
    // One CTA per head up to 8192 rows, eight beyond (a portable cluster); up to 16 rows per thread keys stay in registers.  Measured (us, whole eviction to a
    // quarter, replayed graph, one CTA against eight): 8 heads of 1024 rows 18.0 and 23.5, 2048 18.1 and 23.7, 4096 18.8 and 24.2, 8192 19.9 and 26.2, 16384 27.9 and 32.9
    // (by a sixteenth: 28.1 and 26.3); 128 heads of 1024 rows 26 and 143, 8192 63 and 185, 16384 117 and 246.  Longer slabs would leave a CTA's threads more rows
    // than registers.  (So a CTA alone would serve many heads of up to 16384 rows better; clusters are for few heads of long slabs.)
    const int ranks = a.c.T <= 8192 ? 1 : kRanks, per = rows_per_thread(a.c.T, ranks);
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
    cudaError_t e = cudaLaunchKernelEx(&cfg, per <= 8 ? flb_kv8_select_kernel<8> : per <= 16 ? flb_kv8_select_kernel<16> : flb_kv8_select_kernel<0>, a);
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
