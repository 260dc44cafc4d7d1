// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[m, :] = scale * table[tok[m], :]          zeros where tok[m] is the padding id or out of range
//   gradient  d_table[v, :] = scale * sum over m with tok[m] = v of dy[m, :]
//
// The gradient is a segmented sum.  The token positions are put in the order of their ids by a stable radix sort
// (positions with the same id keep their order), then waves walk fixed-length pieces of the sorted list and keep one
// f32 sum per run of equal ids.  A run inside one piece is written at once; a run over several pieces leaves one
// partial row per piece, and the partial rows are added in the order of the pieces.  Every sum has one fixed order:
// the result depends neither on timing nor on atomics.
#include "row_io.h"

namespace {

// ---- lookup ------------------------------------------------------------------------------------------
// 2^lanes_log2 lanes (at most a wave) share a row.
template <typename TT, typename TO, typename TID, int VEC>
__global__ __launch_bounds__(256) void embedding_kernel(const TID *__restrict__ tokens, const TT *__restrict__ table,
                                                        TO *__restrict__ out, long M, int E, long vocab, float scale,
                                                        long pad_idx, int lanes_log2, int32_t *bad) {
    const int sub = threadIdx.x & ((1 << lanes_log2) - 1);
    const long step = (long)gridDim.x * 256 >> lanes_log2;
    for (long row = ((long)blockIdx.x * 256 + threadIdx.x) >> lanes_log2; row < M; row += step) {
        const long tok = (long)tokens[row];
        const bool pad = tok == pad_idx;
        const bool out_of_range = !pad && (tok < 0 || tok >= vocab);
        if (out_of_range && bad && sub == 0) *bad = 1;
        TO *dst = out + row * E;
        const TT *src = table + (pad || out_of_range ? 0 : tok) * E;
        for (int c = sub * VEC; c < E; c += VEC << lanes_log2) {
            float v[VEC];
            if (pad || out_of_range) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = 0.f;
            } else {
                tc_load_row<TT, VEC>(src + c, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] *= scale;      // in f32, rounded once by the store
            }
            tc_store_row<TO, VEC>(dst + c, v);
        }
    }
}

// ---- stable radix sort of the token positions ------------------------------------------------------------
// Key of a position: its id, or `vocab` (sorts last, ignored by the sums) for padding and ids out of range.
constexpr int kSortTile = 1024;       // positions a workgroup sorts per pass while there are few
constexpr int kMaxBlocks = 256;
constexpr int kMaxBits = 9;

struct SortParams {
    const void *tokens;               // first pass: ids (4 or 8 bytes each)
    const uint32_t *keys_in, *pos_in; // later passes
    uint32_t *keys_out, *pos_out;
    uint32_t *hist;                   // [blocks][bins]
    int id_bytes;                     // 0: keys_in / pos_in
    int M, tile, shift, bits;
    long vocab, pad_idx;
};

__device__ __forceinline__ uint32_t sort_key(const SortParams &p, int i) {
    if (p.id_bytes == 0) return p.keys_in[i];
    const long tok = p.id_bytes == 8 ? static_cast<const long *>(p.tokens)[i] : (long)static_cast<const int32_t *>(p.tokens)[i];
    return tok == p.pad_idx || tok < 0 || tok >= p.vocab ? (uint32_t)p.vocab : (uint32_t)tok;
}

__global__ __launch_bounds__(256) void sort_hist_kernel(const SortParams p) {
    __shared__ uint32_t h[1 << kMaxBits];
    const int bins = 1 << p.bits;
    for (int d = threadIdx.x; d < bins; d += 256) h[d] = 0;
    __syncthreads();
    const int begin = blockIdx.x * p.tile, end = min(p.M, begin + p.tile);
    for (int i = begin + threadIdx.x; i < end; i += 256) atomicAdd(&h[(sort_key(p, i) >> p.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += 256) p.hist[(long)blockIdx.x * bins + d] = h[d];
}

// Where this workgroup's positions of digit d go: all positions of smaller digits, then those of the same digit in
// earlier workgroups, earlier waves of this one, earlier lanes.
__global__ __launch_bounds__(256) void sort_scatter_kernel(const SortParams p) {
    __shared__ uint32_t at[4][1 << kMaxBits];      // next place per wave and digit
    __shared__ uint32_t total[1 << kMaxBits];
    const int bins = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = blockIdx.x * p.tile, end = min(p.M, begin + p.tile);
    const int span = p.tile / 4;                   // tile is a multiple of 256
    const int w_begin = begin + wave * span, w_end = min(end, w_begin + span);
    for (int d = threadIdx.x; d < 4 * bins; d += 256) at[d >> p.bits][d & (bins - 1)] = 0;
    __syncthreads();
    for (int i = w_begin + lane; i < w_end; i += 64) atomicAdd(&at[wave][(sort_key(p, i) >> p.shift) & (bins - 1)], 1u);
    uint32_t before[2] = {0, 0};                   // bins <= 512: at most two digits per thread
    for (int k = 0, d = threadIdx.x; d < bins; d += 256, ++k) {
        uint32_t sum = 0, mine = 0;
#pragma unroll 8
        for (int b = 0; b < (int)gridDim.x; ++b) {
            if (b == (int)blockIdx.x) mine = sum;
            sum += p.hist[(long)b * bins + d];
        }
        total[d] = sum;
        before[k] = mine;
    }
    __syncthreads();
    // exclusive scan of the totals by one wave, eight digits per lane
    if (wave == 0) {
        uint32_t v[8], s = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = lane * 8 + j;
            v[j] = s;
            s += d < bins ? total[d] : 0;
        }
        uint32_t incl = s;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int d = lane * 8 + j;
            if (d < bins) total[d] = incl - s + v[j];
        }
    }
    __syncthreads();
    for (int k = 0, d = threadIdx.x; d < bins; d += 256, ++k) {
        uint32_t place = total[d] + before[k];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t n = at[w][d];
            at[w][d] = place;
            place += n;
        }
    }
    __syncthreads();
    for (int i0 = w_begin; i0 < w_end; i0 += 64) {
        const int i = i0 + lane;
        const bool live = i < w_end;
        const uint32_t key = live ? sort_key(p, i) : 0;
        const uint32_t digit = (key >> p.shift) & (bins - 1);
        unsigned long long same = __ballot(live);
        for (int b = 0; b < p.bits; ++b) {
            const unsigned long long ones = __ballot((digit >> b) & 1u);
            same &= ((digit >> b) & 1u) ? ones : ~ones;
        }
        // the first lane of each digit moves the wave's place on by the number of its lanes
        const int rank = __popcll(same & ((1ull << lane) - 1));
        uint32_t place = 0;
        if (live && rank == 0) place = atomicAdd(&at[wave][digit], (uint32_t)__popcll(same));
        const int first = same ? __ffsll((long long)same) - 1 : 0;
        place = __shfl(place, first, 64) + rank;
        if (live) {
            p.keys_out[place] = key;
            p.pos_out[place] = p.id_bytes ? (uint32_t)i : p.pos_in[i];
        }
    }
}

// ---- segmented sum ----------------------------------------------------------------------------------------
struct SumParams {
    const uint32_t *keys, *pos;       // sorted
    const void *dy;
    long ld_dy;
    float *out;                       // [vocab, E]
    float *partial;                   // [pieces][2][part_ld]: run from the piece before, run into the piece after
    int part_ld;
    int M, E, piece, pieces, accumulate;
    uint32_t vocab;
    float scale;
};

template <int VEC>
__device__ __forceinline__ void write_row(const SumParams &p, uint32_t key, int col, const float (&acc)[VEC]) {
    float v[VEC];
    float *dst = p.out + (long)key * p.E + col;
    if (p.accumulate) {
        tc_load_row<float, VEC>(dst, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] += p.scale * acc[j];
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = p.scale * acc[j];
    }
    tc_store_row<float, VEC>(dst, v);
}

// One wave: one piece of the sorted list (at most 64 positions) x 64 VEC columns.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void segment_sum_kernel(const SumParams p) {
    const int lane = threadIdx.x & 63;
    const int c = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slab = blockIdx.y;
    if (c >= p.pieces) return;
    const int begin = c * p.piece, n = min(p.piece, p.M - begin);
    const int mine = begin + min(lane, n - 1);
    const int keys = (int)p.keys[mine], pos = (int)p.pos[mine];
    const int before = begin > 0 ? (int)p.keys[begin - 1] : -1;
    const int after = begin + n < p.M ? (int)p.keys[begin + n] : -1;
    const int col = slab * 64 * VEC + lane * VEC;
    const bool in = col < p.E;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    int run = 0;                                   // where the current run starts in the piece
    constexpr int U = 8;                           // rows in flight
    for (int i0 = 0; i0 < n; i0 += U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = __builtin_amdgcn_readlane(pos, min(i0 + u, n - 1));
            if (in) tc_load_row<T, VEC>(static_cast<const T *>(p.dy) + (long)(uint32_t)at * p.ld_dy + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u;
            if (i >= n) break;
            const int key = __builtin_amdgcn_readlane(keys, i);
            if ((uint32_t)key == p.vocab) return;  // padding and ids out of range fill the end of the list
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
            const int next = i + 1 < n ? __builtin_amdgcn_readlane(keys, i + 1) : after;
            if (next == key && i + 1 < n) continue;
            const bool from_before = run == 0 && before == key, into_after = next == key;
            if (in) {
                if (!from_before && !into_after) write_row<VEC>(p, (uint32_t)key, col, acc);
                else tc_store_row<float, VEC>(p.partial + ((long)c * 2 + (from_before ? 0 : 1)) * p.part_ld + col, acc);
            }
            run = i + 1;
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        }
    }
}

// Runs over several pieces: the wave of the piece in which the run starts adds the partial rows in order.
template <int VEC>
__global__ __launch_bounds__(256) void segment_join_kernel(const SumParams p) {
    const int lane = threadIdx.x & 63;
    const int c = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slab = blockIdx.y;
    if (c + 1 >= p.pieces) return;
    const int begin = c * p.piece;
    const uint32_t key = p.keys[begin + p.piece - 1];
    if (key == p.vocab || p.keys[begin + p.piece] != key) return;
    if (begin > 0 && p.keys[begin - 1] == key) return;           // starts earlier
    const int col = slab * 64 * VEC + lane * VEC;
    const bool in = col < p.E;
    float acc[VEC], v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (in) tc_load_row<float, VEC>(p.partial + ((long)c * 2 + 1) * p.part_ld + col, acc);
    for (int k = c + 1; k < p.pieces && p.keys[k * p.piece] == key; ++k) {
        if (!in) continue;
        tc_load_row<float, VEC>(p.partial + (long)k * 2 * p.part_ld + col, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[j];
    }
    if (in) write_row<VEC>(p, key, col, acc);
}

__global__ __launch_bounds__(256) void fill_zero_kernel(float *__restrict__ out, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) out[i] = 0.f;
}

struct BwdPlan {
    int tile, blocks, passes, bits, piece, pieces, part_ld;
    size_t keys[2], pos[2], hist, partial, total;
};
BwdPlan bwd_plan(long M, long E, long vocab) {
    BwdPlan w{};
    long tile = (M + kMaxBlocks - 1) / kMaxBlocks;
    tile = (tile + 255) / 256 * 256;
    w.tile = (int)(tile < kSortTile ? kSortTile : tile);
    w.blocks = (int)((M + w.tile - 1) / w.tile);
    int bits = 0;
    while ((vocab >> bits) != 0) ++bits;           // keys 0 .. vocab
    w.passes = (bits + kMaxBits - 1) / kMaxBits;
    w.bits = (bits + w.passes - 1) / w.passes;
    w.piece = 64;
    w.pieces = (int)((M + w.piece - 1) / w.piece);
    w.part_ld = (int)((E + 3) / 4 * 4);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off += (bytes + 255) & ~(size_t)255;
        return o;
    };
    for (int k = 0; k < 2; ++k) { w.keys[k] = take((size_t)M * 4); w.pos[k] = take((size_t)M * 4); }
    w.hist = take((size_t)w.blocks * (1 << w.bits) * 4);
    w.partial = take((size_t)w.pieces * 2 * w.part_ld * 4);
    w.total = off;
    return w;
}

bool embedding_dims_ok(long M, long E, long vocab) {
    return M > 0 && M <= 0x7fffffffL - 1024 && E > 0 && E <= 65536 && vocab > 0 && vocab < 0x7fffffffL;
}

}  // namespace

extern "C" int tc_embedding_fwd(int table_dtype, int out_dtype, int id_bytes, const void *tokens, const void *table,
                                void *out, long M, int E, long vocab, float scale, long pad_idx, int32_t *bad,
                                void *stream) {
    TC_REQUIRE(tokens && table && out, "tc_embedding_fwd: null operand");
    TC_REQUIRE((table_dtype == TC_F32 || table_dtype == TC_BF16) && (out_dtype == TC_F32 || out_dtype == TC_BF16),
               "tc_embedding_fwd: bad dtype");
    TC_REQUIRE(id_bytes == 4 || id_bytes == 8, "tc_embedding_fwd: ids of %d bytes (4 or 8)", id_bytes);
    TC_REQUIRE(embedding_dims_ok(M, E, vocab), "tc_embedding_fwd: bad shape M=%ld E=%d vocab=%ld", M, E, vocab);
    const int t_esz = table_dtype == TC_BF16 ? 2 : 4, o_esz = out_dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE((uintptr_t)table % t_esz == 0 && (uintptr_t)out % o_esz == 0 && (uintptr_t)tokens % id_bytes == 0,
               "tc_embedding_fwd: misaligned operand");
    if (pad_idx < 0) pad_idx = INT64_MIN;          // no padding id
    // 16-byte stores where the rows allow them: 4 f32 or 8 bf16 values
    const int wide = out_dtype == TC_BF16 ? 8 : 4;
    const bool vec = tc_rows_aligned(table, E, t_esz, wide) && tc_rows_aligned(out, E, o_esz, wide);
    const int pieces = vec ? E / wide : E;
    int lanes_log2 = 0;
    while (lanes_log2 < 6 && (1 << lanes_log2) < pieces) ++lanes_log2;
    long blocks = ((M << lanes_log2) + 255) / 256;
    if (blocks > (1L << 20)) blocks = 1L << 20;    // a launch holds fewer than 2^32 threads; rows are walked with the grid's stride
    hipStream_t s = static_cast<hipStream_t>(stream);
    TcProfScope prof(TC_PROF_EMBED, s, (double)M * E * o_esz);
#define TC_EMB(TT, TO, TID, V)                                                                              \
    TC_LAUNCH((embedding_kernel<TT, TO, TID, V>), dim3((unsigned)blocks), dim3(256), 0, s,                  \
              static_cast<const TID *>(tokens), static_cast<const TT *>(table), static_cast<TO *>(out), M, E, vocab, scale, \
              pad_idx, lanes_log2, bad)
#define TC_EMB_ID(TT, TO, V) do { if (id_bytes == 4) TC_EMB(TT, TO, int32_t, V); else TC_EMB(TT, TO, int64_t, V); } while (0)
#define TC_EMB_V(TT, TO, W) do { if (vec) TC_EMB_ID(TT, TO, W); else TC_EMB_ID(TT, TO, 1); } while (0)
    if (table_dtype == TC_F32) {
        if (out_dtype == TC_F32) TC_EMB_V(float, float, 4);
        else TC_EMB_V(float, uint16_t, 8);
    } else {
        if (out_dtype == TC_F32) TC_EMB_V(uint16_t, float, 4);
        else TC_EMB_V(uint16_t, uint16_t, 8);
    }
#undef TC_EMB_V
#undef TC_EMB_ID
#undef TC_EMB
    TC_CHECK_LAUNCH("tc_embedding_fwd");
    return TC_OK;
}

extern "C" size_t tc_embedding_bwd_workspace_bytes(long M, int E, long vocab) {
    return embedding_dims_ok(M, E, vocab) ? bwd_plan(M, E, vocab).total : 0;
}

extern "C" int tc_embedding_bwd(int dy_dtype, int id_bytes, const void *tokens, const void *dy, long ld_dy, float *d_table,
                                long M, int E, long vocab, float scale, long pad_idx, int accumulate, void *workspace,
                                size_t workspace_bytes, void *stream) {
    TC_REQUIRE(tokens && dy && d_table && workspace, "tc_embedding_bwd: null operand");
    TC_REQUIRE(dy_dtype == TC_F32 || dy_dtype == TC_BF16, "tc_embedding_bwd: bad dtype %d", dy_dtype);
    TC_REQUIRE(id_bytes == 4 || id_bytes == 8, "tc_embedding_bwd: ids of %d bytes (4 or 8)", id_bytes);
    TC_REQUIRE(embedding_dims_ok(M, E, vocab) && ld_dy >= E, "tc_embedding_bwd: bad shape M=%ld E=%d vocab=%ld ld=%ld", M, E,
               vocab, ld_dy);
    const int esz = dy_dtype == TC_BF16 ? 2 : 4;
    TC_REQUIRE((uintptr_t)dy % esz == 0 && (uintptr_t)d_table % 4 == 0 && (uintptr_t)tokens % id_bytes == 0 &&
                   tc_aligned16(workspace),
               "tc_embedding_bwd: misaligned operand");
    const BwdPlan w = bwd_plan(M, E, vocab);
    if (workspace_bytes < w.total) {
        tc_set_error("tc_embedding_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, w.total);
        return TC_ENOSPC;
    }
    if (pad_idx < 0) pad_idx = INT64_MIN;
    char *ws = static_cast<char *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    SortParams sp{};
    sp.tokens = tokens;
    sp.id_bytes = id_bytes;
    sp.M = (int)M; sp.tile = w.tile; sp.bits = w.bits;
    sp.vocab = vocab; sp.pad_idx = pad_idx;
    sp.hist = reinterpret_cast<uint32_t *>(ws + w.hist);
    for (int pass = 0; pass < w.passes; ++pass) {
        sp.shift = pass * w.bits;
        sp.keys_out = reinterpret_cast<uint32_t *>(ws + w.keys[pass & 1]);
        sp.pos_out = reinterpret_cast<uint32_t *>(ws + w.pos[pass & 1]);
        TC_LAUNCH(sort_hist_kernel, dim3(w.blocks), dim3(256), 0, s, sp);
        TC_LAUNCH(sort_scatter_kernel, dim3(w.blocks), dim3(256), 0, s, sp);
        sp.id_bytes = 0;
        sp.keys_in = sp.keys_out;
        sp.pos_in = sp.pos_out;
    }
    SumParams q{};
    q.keys = sp.keys_in; q.pos = sp.pos_in;
    q.dy = dy; q.ld_dy = ld_dy;
    q.out = d_table;
    q.partial = reinterpret_cast<float *>(ws + w.partial);
    q.part_ld = w.part_ld;
    q.M = (int)M; q.E = E; q.piece = w.piece; q.pieces = w.pieces;
    q.accumulate = accumulate; q.vocab = (uint32_t)vocab; q.scale = scale;
    const bool vec = tc_rows_aligned(dy, ld_dy, esz, 4) && tc_rows_aligned(d_table, E, 4, 4);
    const dim3 blocks((w.pieces + 3) / 4, (E + (vec ? 255 : 63)) / (vec ? 256 : 64));
    if (!accumulate) {
        const long n = vocab * E;
        const long most = 4096;
        TC_LAUNCH(fill_zero_kernel, dim3((unsigned)((n + 255) / 256 < most ? (n + 255) / 256 : most)), dim3(256), 0, s, d_table, n);
    }
    if (dy_dtype == TC_F32) {
        if (vec) TC_LAUNCH((segment_sum_kernel<float, 4>), blocks, dim3(256), 0, s, q);
        else TC_LAUNCH((segment_sum_kernel<float, 1>), blocks, dim3(256), 0, s, q);
    } else {
        if (vec) TC_LAUNCH((segment_sum_kernel<uint16_t, 4>), blocks, dim3(256), 0, s, q);
        else TC_LAUNCH((segment_sum_kernel<uint16_t, 1>), blocks, dim3(256), 0, s, q);
    }
    if (w.pieces > 1) {
        if (vec) TC_LAUNCH(segment_join_kernel<4>, blocks, dim3(256), 0, s, q);
        else TC_LAUNCH(segment_join_kernel<1>, blocks, dim3(256), 0, s, q);
    }
    TC_CHECK_LAUNCH("tc_embedding_bwd");
    return TC_OK;
}
