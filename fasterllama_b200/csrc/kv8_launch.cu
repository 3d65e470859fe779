// kv8_launch.cu — the extern "C" layer declared in include/flb_kv8.h: argument checks, scratch carving, launches.
// Stream-ordered, allocation-free, no synchronisation, no exit(), no exceptions.
#include "../../include/flb_kv8.h"
#include "kv8.cuh"

namespace {

inline size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
template <typename... P> inline bool aligned4(const void *p, P... more) { return aligned4(p) && aligned4(more...); }

int check_sizes(const flb_kv8_cache &c) {
    if (c.batch_size <= 0 || c.kv_head_num <= 0 || c.size_per_head <= 0 || c.total_len <= 0) return FLB_ERR_BAD_SHAPE;
    if (c.size_per_head != 64 && c.size_per_head != 128 && c.size_per_head != 256) return FLB_ERR_UNSUPPORTED;
    if (c.block_len != 16 && c.block_len != 32 && c.block_len != 64 && c.block_len != 128) return FLB_ERR_UNSUPPORTED;
    if (c.total_len % c.block_len) return FLB_ERR_BAD_SHAPE;
    if ((size_t)c.batch_size * c.kv_head_num > (size_t)1 << 24) return FLB_ERR_TOO_LARGE;
    if (c.total_len > 1 << 30) return FLB_ERR_TOO_LARGE; // row arithmetic in int
    if ((size_t)c.kv_head_num * c.size_per_head > 0x7fffffffu) return FLB_ERR_TOO_LARGE; // so are row strides
    return FLB_OK;
}
int check_cache(const flb_kv8_cache &c) {
    const int st = check_sizes(c);
    if (st != FLB_OK) return st;
    if (c.code_type != FLB_KV8_I8 && c.code_type != FLB_KV8_E4M3) return FLB_ERR_BAD_ENUM;
    if (!c.k_codes || !c.v_codes || !c.k_scale || !c.v_scale) return FLB_ERR_NULL_POINTER;
    if (!aligned16(c.k_codes) || !aligned16(c.v_codes)) return FLB_ERR_MISALIGNED;
    if (!aligned4(c.k_scale, c.v_scale, c.row_pos)) return FLB_ERR_MISALIGNED;
    return FLB_OK;
}
// one of q, k, v: pointer, scale, stride (elements; 0 = dense)
int check_input(int mode, const void *p, const float *w_scale, int stride, int dense) {
    if (!p) return FLB_ERR_NULL_POINTER;
    if (mode == FLB_IN_INT32 && !w_scale) return FLB_ERR_NULL_POINTER;
    if (!aligned16(p) || (mode == FLB_IN_INT32 && !aligned16(w_scale))) return FLB_ERR_MISALIGNED;
    if (stride != 0) {
        if (stride < dense) return FLB_ERR_BAD_SHAPE;
        if (((size_t)stride * (mode == FLB_IN_F16 ? 2 : 4)) % 16u) return FLB_ERR_MISALIGNED;
    }
    return FLB_OK;
}
int check_rope(const float *freq_cis, int rows) {
    if (!freq_cis) return FLB_OK;
    if (rows <= 0) return FLB_ERR_BAD_SHAPE;
    return aligned16(freq_cis) ? FLB_OK : FLB_ERR_MISALIGNED;
}

flb::Kv8Cache cache_of(const flb_kv8_cache &c) {
    flb::Kv8Cache k;
    k.B = c.batch_size;
    k.H = c.kv_head_num;
    k.T = c.total_len;
    k.block_shift = 4;
    while ((1 << k.block_shift) < c.block_len) ++k.block_shift;
    k.nblk = c.total_len / c.block_len;
    k.codes[0] = static_cast<uint8_t *>(c.k_codes);
    k.codes[1] = static_cast<uint8_t *>(c.v_codes);
    k.scale[0] = c.k_scale;
    k.scale[1] = c.v_scale;
    k.row_pos = c.row_pos;
    return k;
}

// blocks that S tokens behind any number of cached rows can touch
inline int window_blocks(const flb_kv8_cache &c, int S, bool any_past, int start) {
    const int bl = c.block_len;
    const int n = any_past ? (S - 2 + bl) / bl + 1 : (start + S - 1) / bl - start / bl + 1;
    return n < c.total_len / bl ? n : c.total_len / bl;
}

// Rows of one split when the caller names none: a function of the slab's capacity alone, so results stay the same under any sharding of
// the batch and the heads.  A CTA costs about 3 us besides its rows, of which four per SM overlap, and every split a partial result.  Measured
// (us, replayed graph; 16 x 32 heads of 1024-2047 rows): 256 rows 48.2, 512 41.3, 1024 43.4, 2048 39.8; (1 x 32 heads, 1000 rows) 8.5, 9.5, 9.8; (1 x 8
// heads of 4 q heads, 8000 rows) 9.9, 9.9, 13.8, 18.7; (the same, 100001 rows) 72, 55, 51, 42.
inline int split_len_of(const flb_kv8_decode_params *p) {
    if (p->split_len > 0) return p->split_len;
    const int T = p->cache.total_len;
    return T <= 512 ? 256 : T <= 8192 ? 512 : T <= 32768 ? 1024 : 2048;
}
inline int max_past_of(const flb_kv8_decode_params *p) {
    if (!p->past_lens) return p->start_pos;
    return p->max_past_len > 0 ? p->max_past_len : p->cache.total_len - 1;
}

// q heads of one K/V head are dealt out over CTAs of 4 or 8: 8 from five heads on (d = 256: registers hold 4)
struct HeadSplit {
    int nt, nchunk;
};
inline HeadSplit heads_for(int G, int d) {
    HeadSplit s;
    s.nt = (G > 4 && d != 256) ? 2 : 1;
    s.nchunk = (G + 4 * s.nt - 1) / (4 * s.nt);
    return s;
}

struct DecodeScratch {
    size_t counter_bytes, ml_off, o_off, fml_off, score_off, total;
};
DecodeScratch decode_scratch(const flb_kv8_decode_params *p, int max_past, bool weights) {
    DecodeScratch l;
    const size_t units = (size_t)p->cache.batch_size * p->cache.kv_head_num;
    const HeadSplit hs = heads_for(p->head_num / p->cache.kv_head_num, p->cache.size_per_head);
    const size_t nsplit = (size_t)max_past / split_len_of(p) + 1;
    const size_t parts = units * hs.nchunk * nsplit * 4 * hs.nt;
    l.counter_bytes = round_up(sizeof(unsigned) * (4 + units * hs.nchunk), 256);
    l.ml_off = l.counter_bytes;
    l.o_off = l.ml_off + round_up(parts * 2 * sizeof(float), 256);
    l.fml_off = l.o_off + round_up(parts * p->cache.size_per_head * sizeof(float), 256);
    const size_t heads = (size_t)p->cache.batch_size * p->head_num;
    l.score_off = l.fml_off + (weights ? round_up(heads * 2 * sizeof(float), 256) : 0);
    l.total = l.score_off + (weights ? heads * p->cache.total_len * sizeof(float) : 0);
    return l;
}

int check_decode_sizes(const flb_kv8_decode_params *p) {
    const int st = check_sizes(p->cache);
    if (st != FLB_OK) return st;
    if (p->head_num <= 0 || p->head_num % p->cache.kv_head_num) return FLB_ERR_BAD_SHAPE;
    if (p->split_len < 0 || p->split_len % 128 || p->split_len > 2048) return FLB_ERR_BAD_SHAPE;
    if ((size_t)p->cache.batch_size * p->head_num > (size_t)1 << 24 || (size_t)p->head_num * p->cache.size_per_head > 0x7fffffffu) return FLB_ERR_TOO_LARGE;
    return FLB_OK;
}

size_t evict_bytes(const flb_kv8_cache &c) {
    const size_t units = (size_t)c.batch_size * c.kv_head_num;
    return 256 + round_up((size_t)c.batch_size * 2 * sizeof(int), 256) + round_up(units * 2 * sizeof(float), 256) + round_up(units * (c.total_len / c.block_len + 1) * sizeof(int), 256) +
           2 * round_up(units * (c.total_len / 2) * sizeof(int), 256); // a hole has a source: at most half the rows are either
}

} // namespace

extern "C" {

int flb_kv8_validate_append(const flb_kv8_append_params *p) {
    if (!p) return FLB_ERR_NULL_POINTER;
    int st = check_cache(p->cache);
    if (st != FLB_OK) return st;
    if (p->seq_len <= 0 || p->seq_len > p->cache.total_len) return FLB_ERR_BAD_SHAPE;
    if (p->input_mode < FLB_IN_INT32 || p->input_mode > FLB_IN_F16) return FLB_ERR_BAD_ENUM;
    if (p->input_mode == FLB_IN_INT32 && !p->act_scale) return FLB_ERR_NULL_POINTER;
    const int dense = p->cache.kv_head_num * p->cache.size_per_head;
    if ((st = check_input(p->input_mode, p->k, p->k_w_scale, p->kv_row_stride, dense)) != FLB_OK) return st;
    if ((st = check_input(p->input_mode, p->v, p->v_w_scale, p->kv_row_stride, dense)) != FLB_OK) return st;
    if ((st = check_rope(p->freq_cis, p->freq_rows)) != FLB_OK) return st;
    if (!aligned4(p->past_lens, p->new_lens, p->token_pos, p->act_scale, p->status)) return FLB_ERR_MISALIGNED;
    if (!p->past_lens && (p->start_pos < 0 || p->start_pos > p->cache.total_len - p->seq_len)) return FLB_ERR_BAD_SHAPE;
    // one CTA per block that a call can touch: the grid's second and third extents hold 65535
    if (p->cache.batch_size > 65535 || window_blocks(p->cache, p->seq_len, p->past_lens != nullptr, p->start_pos) > 65535) return FLB_ERR_TOO_LARGE;
    return FLB_OK;
}

int flb_kv8_validate_decode(const flb_kv8_decode_params *p) {
    if (!p) return FLB_ERR_NULL_POINTER;
    int st = check_cache(p->cache);
    if (st != FLB_OK) return st;
    if ((st = check_decode_sizes(p)) != FLB_OK) return st;
    if (p->input_mode < FLB_IN_INT32 || p->input_mode > FLB_IN_F16) return FLB_ERR_BAD_ENUM;
    if (p->out_dtype != FLB_F32 && p->out_dtype != FLB_F16) return FLB_ERR_BAD_ENUM;
    if (p->input_mode == FLB_IN_INT32 && !p->act_scale) return FLB_ERR_NULL_POINTER;
    const int d = p->cache.size_per_head;
    if ((st = check_input(p->input_mode, p->q, p->q_w_scale, p->q_row_stride, p->head_num * d)) != FLB_OK) return st;
    if ((st = check_input(p->input_mode, p->k, p->k_w_scale, p->kv_row_stride, p->cache.kv_head_num * d)) != FLB_OK) return st;
    if ((st = check_input(p->input_mode, p->v, p->v_w_scale, p->kv_row_stride, p->cache.kv_head_num * d)) != FLB_OK) return st;
    if ((st = check_rope(p->freq_cis, p->freq_rows)) != FLB_OK) return st;
    if (!flb::cap_ok(p->softcap)) return FLB_ERR_BAD_SHAPE;
    if (!p->out) return FLB_ERR_NULL_POINTER;
    if (!aligned16(p->out)) return FLB_ERR_MISALIGNED;
    if ((p->weight_in != nullptr) != (p->weight_out != nullptr)) return FLB_ERR_NULL_POINTER;
    if (!aligned16(p->weight_in) || !aligned16(p->weight_out)) return FLB_ERR_MISALIGNED;
    if (!aligned4(p->past_lens, p->token_pos, p->act_scale, p->alibi_slopes, p->key_begin)) return FLB_ERR_MISALIGNED;
    const int mp = max_past_of(p);
    if (mp < 0 || mp >= p->cache.total_len) return FLB_ERR_BAD_SHAPE;
    if (!p->scratch) return FLB_ERR_NULL_POINTER;
    if (!aligned16(p->scratch)) return FLB_ERR_MISALIGNED;
    const HeadSplit hs = heads_for(p->head_num / p->cache.kv_head_num, d);
    const unsigned long long units = (unsigned long long)p->cache.batch_size * p->cache.kv_head_num;
    if (units * hs.nchunk * (mp / split_len_of(p) + 1) > 0x7fffffffull || units * (mp / 1024 + 2) > 0x7fffffffull) return FLB_ERR_TOO_LARGE;
    if (hs.nchunk > 1 && p->cache.batch_size > 65535) return FLB_ERR_TOO_LARGE; // the append in front has a grid extent of that many
    if (p->scratch_bytes < decode_scratch(p, mp, p->weight_out != nullptr).total) return FLB_ERR_SCRATCH_TOO_SMALL;
    return FLB_OK;
}

int flb_kv8_validate_evict(const flb_kv8_evict_params *p) {
    if (!p) return FLB_ERR_NULL_POINTER;
    const int st = check_cache(p->cache);
    if (st != FLB_OK) return st;
    if (!p->cache.row_pos || !p->len_out || !p->weight || !p->weight_out || !p->pos_out || !p->scratch) return FLB_ERR_NULL_POINTER;
    if (p->recent > 0 && !p->next_pos) return FLB_ERR_NULL_POINTER;
    if (p->budget <= 0 || p->recent < 0 || p->sinks < 0 || p->recent > p->budget || p->sinks > p->budget - p->recent) return FLB_ERR_BAD_SHAPE;
    if (!p->past_lens && (p->start_pos < 0 || p->start_pos > p->cache.total_len)) return FLB_ERR_BAD_SHAPE;
    if (!aligned16(p->scratch) || !aligned4(p->past_lens, p->len_out, p->next_pos)) return FLB_ERR_MISALIGNED;
    if (!aligned16(p->weight) || !aligned16(p->cache.row_pos) || !aligned16(p->weight_out) || !aligned16(p->pos_out)) return FLB_ERR_MISALIGNED;
    if (8ull * p->cache.batch_size * p->cache.kv_head_num * (p->cache.total_len / p->cache.block_len + 1) > 0x7fffffffull) return FLB_ERR_TOO_LARGE;
    if (p->scratch_bytes < evict_bytes(p->cache)) return FLB_ERR_SCRATCH_TOO_SMALL;
    return FLB_OK;
}

int flb_kv8_decode_workspace_bytes(const flb_kv8_decode_params *p, size_t *bytes_out) {
    if (!p || !bytes_out) return FLB_ERR_NULL_POINTER;
    const int st = check_decode_sizes(p);
    if (st != FLB_OK) return st;
    *bytes_out = decode_scratch(p, p->cache.total_len - 1, p->weight_out != nullptr).total;
    return FLB_OK;
}

int flb_kv8_counter_bytes(const flb_kv8_decode_params *p, size_t *bytes_out) {
    if (!p || !bytes_out) return FLB_ERR_NULL_POINTER;
    const int st = check_decode_sizes(p);
    if (st != FLB_OK) return st;
    *bytes_out = decode_scratch(p, 0, false).counter_bytes;
    return FLB_OK;
}

int flb_kv8_evict_workspace_bytes(const flb_kv8_evict_params *p, size_t *bytes_out) {
    if (!p || !bytes_out) return FLB_ERR_NULL_POINTER;
    const int st = check_sizes(p->cache);
    if (st != FLB_OK) return st;
    *bytes_out = evict_bytes(p->cache);
    return FLB_OK;
}

int flb_kv8_append(const flb_kv8_append_params *p, void *cuda_stream) {
    const int st = flb_kv8_validate_append(p);
    if (st != FLB_OK) return st;
    flb::Kv8AppendArgs a;
    a.c = cache_of(p->cache);
    a.S = p->seq_len;
    a.nwin = window_blocks(p->cache, p->seq_len, p->past_lens != nullptr, p->start_pos);
    a.max_past = p->cache.total_len;
    a.start_pos = p->start_pos;
    a.past_lens = p->past_lens;
    a.new_lens = p->new_lens;
    a.token_pos = p->token_pos;
    const int stride = p->kv_row_stride ? p->kv_row_stride : p->cache.kv_head_num * p->cache.size_per_head;
    a.in[0] = {p->k, p->k_w_scale, stride};
    a.in[1] = {p->v, p->v_w_scale, stride};
    a.act_scale = p->act_scale;
    a.freq_cis = p->freq_cis;
    a.freq_rows = p->freq_rows;
    a.status = p->status;
    return flb::launch_kv8_append(a, p->cache.size_per_head, p->cache.code_type, p->input_mode, static_cast<cudaStream_t>(cuda_stream)) == cudaSuccess
               ? FLB_OK
               : FLB_ERR_LAUNCH;
}

int flb_kv8_decode(const flb_kv8_decode_params *p, void *cuda_stream) {
    const int st = flb_kv8_validate_decode(p);
    if (st != FLB_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const bool weights = p->weight_out != nullptr;
    const int mp = max_past_of(p), d = p->cache.size_per_head, G = p->head_num / p->cache.kv_head_num;
    const DecodeScratch l = decode_scratch(p, mp, weights);
    const HeadSplit hs = heads_for(G, d);
    unsigned char *sc = static_cast<unsigned char *>(p->scratch);
    if (!p->scratch_zeroed && cudaMemsetAsync(sc, 0, l.counter_bytes, stream) != cudaSuccess) return FLB_ERR_LAUNCH;

    flb::Kv8DecodeArgs a;
    a.c = cache_of(p->cache);
    a.input_mode = p->input_mode;
    a.Hq = p->head_num;
    a.G = G;
    a.nchunk = hs.nchunk;
    a.start_pos = p->start_pos;
    a.past_lens = p->past_lens;
    a.token_pos = p->token_pos;
    const int kv_stride = p->kv_row_stride ? p->kv_row_stride : p->cache.kv_head_num * d;
    a.in[0] = {p->q, p->q_w_scale, p->q_row_stride ? p->q_row_stride : p->head_num * d};
    a.in[1] = {p->k, p->k_w_scale, kv_stride};
    a.in[2] = {p->v, p->v_w_scale, kv_stride};
    a.act_scale = p->act_scale;
    a.freq_cis = p->freq_cis;
    a.freq_rows = p->freq_rows;
    a.scale_log2e = p->softmax_scale * 1.4426950408889634f;
    a.cap_log2e = p->softcap * 1.4426950408889634f;
    a.slopes = p->alibi_slopes;
    a.key_begin = p->key_begin;
    a.scores = weights ? reinterpret_cast<float *>(sc + l.score_off) : nullptr;
    a.ml = weights ? reinterpret_cast<float *>(sc + l.fml_off) : nullptr;
    a.weight_in = p->weight_in;
    a.weight_out = p->weight_out;
    a.out = p->out;
    a.out_f16 = p->out_dtype == FLB_F16;
    a.append = hs.nchunk == 1;
    a.split_len = split_len_of(p);
    a.max_past = mp; // below the slab's capacity
    a.nsplit_max = mp / a.split_len + 1;
    a.status = reinterpret_cast<unsigned *>(sc);
    a.counters = reinterpret_cast<unsigned *>(sc) + 4;
    a.part_ml = reinterpret_cast<float *>(sc + l.ml_off);
    a.part_o = reinterpret_cast<float *>(sc + l.o_off);
    if (!a.append) {
        flb::Kv8AppendArgs t;
        t.c = a.c;
        t.S = 1;
        t.nwin = 1;
        t.max_past = mp; // what the attention kernel will not look at is not stored either
        t.start_pos = a.start_pos;
        t.past_lens = a.past_lens;
        t.new_lens = nullptr;
        t.token_pos = a.token_pos;
        t.in[0] = a.in[1];
        t.in[1] = a.in[2];
        t.act_scale = a.act_scale;
        t.freq_cis = a.freq_cis;
        t.freq_rows = a.freq_rows;
        t.status = a.status;
        if (flb::launch_kv8_append(t, d, p->cache.code_type, p->input_mode, stream) != cudaSuccess) return FLB_ERR_LAUNCH;
    }
    return flb::launch_kv8_decode(a, d, p->cache.code_type, hs.nt, stream) == cudaSuccess ? FLB_OK : FLB_ERR_LAUNCH;
}

int flb_kv8_evict(const flb_kv8_evict_params *p, void *cuda_stream) {
    const int st = flb_kv8_validate_evict(p);
    if (st != FLB_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const size_t units = (size_t)p->cache.batch_size * p->cache.kv_head_num, T = p->cache.total_len;
    unsigned char *sc = static_cast<unsigned char *>(p->scratch);
    flb::Kv8EvictArgs a;
    a.c = cache_of(p->cache);
    a.start_pos = p->start_pos;
    a.past_lens = p->past_lens;
    a.len_out = p->len_out;
    a.budget = p->budget;
    a.recent = p->recent;
    a.sinks = p->sinks;
    a.next_pos = p->next_pos;
    a.weight = p->weight;
    a.weight_out = p->weight_out;
    a.pos_out = p->pos_out;
    a.status = reinterpret_cast<unsigned *>(sc);
    size_t o = 256;
    a.seq_len = reinterpret_cast<int *>(sc + o);
    o += round_up((size_t)p->cache.batch_size * 2 * sizeof(int), 256);
    a.edge_scale = reinterpret_cast<float *>(sc + o);
    o += round_up(units * 2 * sizeof(float), 256);
    a.hole_off = reinterpret_cast<int *>(sc + o);
    o += round_up(units * (a.c.nblk + 1) * sizeof(int), 256);
    a.moves = reinterpret_cast<int *>(sc + o);
    o += round_up(units * (T / 2) * sizeof(int), 256);
    a.holes = reinterpret_cast<int *>(sc + o);
    return flb::launch_kv8_evict(a, p->cache.size_per_head, p->cache.code_type, stream) == cudaSuccess ? FLB_OK : FLB_ERR_LAUNCH;
}

} // extern "C"
