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
template <typename TT, typename TO, typename TID, int VEC, bool LOOSE>
__global__ __launch_bounds__(256) void embedding_kernel(const TID *__restrict__ tokens, const TT *__restrict__ table,
                                                        TO *__restrict__ out, long M, int E, long vocab, float scale,
                                                        long pad_idx, int lanes_log2, int32_t *bad) {
    const int sub = threadIdx.x & ((1 << lanes_log2) - 1);
    const long step = (long)gridDim.x * 256 >> lanes_log2;
    for (long row = ((long)blockIdx.x * 256 + threadIdx.x) >> lanes_log2; row < M; row += step) {
        const long tok = (long)tokens[row];
        const bool pad = pad_idx >= 0 && tok == pad_idx;      // no id below 0 is padding, whatever pad_idx is
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
                tc_load_row<TT, VEC, LOOSE>(src + c, v, E - c);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] *= scale;      // in f32, rounded once by the store
            }
            tc_store_row<TO, VEC, LOOSE>(dst + c, v, E - c);
        }
    }
}

// Columns of a lane in the gradient's kernels; a wave takes 64 VEC.  (8 of bf16, one 16-byte load, halves the waves: 47 instead
// of 39 us for the sums of 49153 x 1024.)
constexpr int VEC = 4;

// ---- gradient of a few positions -----------------------------------------------------------------------
// Up to kFew positions: no sort.  Every wave holds all ids, finds the positions of a table row by comparing, and adds their
// rows of dy in order; rows without a position are written as zeros on the way.
constexpr int kFew = 512;
struct FewParams {
    const void *tokens, *dy;
    float *out;
    long ld_dy, vocab, pad_idx;
    int M, E, accumulate;
    float scale;
};
template <typename T, typename TID, bool LOOSE>
__global__ __launch_bounds__(256) void few_positions_kernel(const FewParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = blockIdx.y * 64 * VEC + lane * VEC;
    const bool in = col < p.E;
    long id[kFew / 64];
#pragma unroll
    for (int k = 0; k < kFew / 64; ++k) {
        const int i = k * 64 + lane;
        id[k] = i < p.M ? (long)static_cast<const TID *>(p.tokens)[i] : -1;
        if (id[k] == p.pad_idx) id[k] = -1;
    }
    for (long v = (long)blockIdx.x * 4 + wave; v < p.vocab; v += (long)gridDim.x * 4) {
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        bool any = false;
#pragma unroll
        for (int k = 0; k < kFew / 64; ++k) {
            unsigned long long left = __ballot(id[k] == v);
            any |= left != 0;
            // U rows in flight; a spent mask repeats its last row
            auto batch = [&](auto u_c) {
                constexpr int U = decltype(u_c)::value;
                int at[U], n = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (left) {
                        at[u] = __ffsll((long long)left) - 1;
                        left &= left - 1;
                        n = u + 1;
                    } else {
                        at[u] = at[u > 0 ? u - 1 : 0];
                    }
                }
                float x[U][VEC];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (in) tc_load_row<T, VEC, LOOSE>(static_cast<const T *>(p.dy) + (long)(k * 64 + at[u]) * p.ld_dy + col, x[u], p.E - col);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u < n)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) acc[j] += x[u][j];
            };
            while (left) {
                if (__popcll(left) > 4) batch(std::integral_constant<int, 16>{});
                else batch(std::integral_constant<int, 4>{});
            }
        }
        if (!in || (p.accumulate && !any)) continue;
        float *dst = p.out + v * p.E + col, old[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) old[j] = 0.f;
        if (p.accumulate) tc_load_row<float, VEC, LOOSE>(dst, old, p.E - col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = any ? old[j] + p.scale * acc[j] : 0.f;      // zero for any scale
        tc_store_row<float, VEC, LOOSE>(dst, acc, p.E - col);
    }
}

// ---- stable radix sort of the token positions ------------------------------------------------------------
// Key of a position: its id, or `vocab` (sorts last, ignored by the sums) for padding and ids out of range.  Digits of at
// most 9 bits from the lowest up; per digit one launch counts every workgroup's positions and a second places them behind
// all smaller digits and all earlier equal ones.  (Counting the next digit with atomics while the present one is placed
// saves a launch, but frequent ids meet on one counter: 65 us instead of 10 at 49153 positions.)  Up to 8192 positions are
// sorted by one workgroup in LDS, all digits in one launch.  The sort keeps few CUs busy, so its launches also clear the gradient,
// a slice each, with workgroups of their own.
constexpr int kSortWaves = 16;
constexpr int kSortThreads = 64 * kSortWaves;
constexpr int kMaxBits = 9;
constexpr int kFewBlocks = 128;

struct SortParams {
    const void *tokens;               // first pass: ids (4 or 8 bytes each)
    uint32_t *keys[2], *pos[2];       // later passes: from [(pass - 1) & 1] to [pass & 1]
    uint32_t *hist;                   // [blocks][bins]
    uint32_t *totals;                 // [bins], with hist already summed over the workgroups before (null: not yet)
    int id_bytes, M, blocks, bits, passes;
    long vocab, pad_idx;
    float *clear;                     // gradient to clear (null: none), this launch's slice
    long clear_from, clear_to;
};

__device__ __forceinline__ uint32_t sort_key(const SortParams &p, int pass, int i) {
    if (pass > 0) return p.keys[(pass - 1) & 1][i];
    const long tok = p.id_bytes == 8 ? static_cast<const long *>(p.tokens)[i] : (long)static_cast<const int32_t *>(p.tokens)[i];
    return tok == p.pad_idx || tok < 0 || tok >= p.vocab ? (uint32_t)p.vocab : (uint32_t)tok;
}

// true for the workgroups behind the sorting ones, after they have cleared their part
__device__ __forceinline__ bool clear_slice(const SortParams &p) {
    if ((int)blockIdx.x < p.blocks) return false;
    const long n = p.clear_to - p.clear_from, step = (long)(gridDim.x - p.blocks) * kSortThreads;
    float *out = p.clear + p.clear_from;
    const long first = (long)(blockIdx.x - p.blocks) * kSortThreads + threadIdx.x;
    if (((uintptr_t)out & 15) == 0) {
        for (long i = first; i < n / 4; i += step) *reinterpret_cast<f32x4 *>(out + 4 * i) = f32x4{0.f, 0.f, 0.f, 0.f};
        for (long i = n / 4 * 4 + first; i < n; i += step) out[i] = 0.f;
    } else {
        for (long i = first; i < n; i += step) out[i] = 0.f;
    }
    return true;
}

// Adds the digits of a wave's lanes, R rounds of them, to its counts, one atomic for all lanes of a digit and round (padding
// would put all 64 on one counter); earlier[r]: how many of the wave's positions before, in order of rounds and lanes, have
// the lane's digit.  Three loops, so that the atomics of all rounds are under way together.
template <int R>
__device__ __forceinline__ void count_digits(const bool (&live)[R], const uint32_t (&digit)[R], uint32_t *counts, int bits,
                                             uint32_t (&earlier)[R]) {
    const int lane = threadIdx.x & 63;
    unsigned long long same[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        same[r] = __ballot(live[r]);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long ones = __ballot((digit[r] >> b) & 1u);
            same[r] &= ((digit[r] >> b) & 1u) ? ones : ~ones;
        }
    }
    uint32_t old[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        old[r] = 0;
        if (live[r] && (same[r] & ((1ull << lane) - 1)) == 0) old[r] = atomicAdd(counts + digit[r], (uint32_t)__popcll(same[r]));
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        earlier[r] = __shfl(old[r], same[r] ? __ffsll((long long)same[r]) - 1 : 0, 64) + __popcll(same[r] & ((1ull << lane) - 1));
}

// Exclusive sums of total[0 .. bins) in place by one wave, at most eight digits a lane.
__device__ __forceinline__ void scan_totals(uint32_t *total, int bins) {
    const int lane = threadIdx.x & 63;
    uint32_t v[8], s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = s;
        s += lane * 8 + j < bins ? total[lane * 8 + j] : 0;
    }
    uint32_t incl = s;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane * 8 + j < bins) total[lane * 8 + j] = incl - s + v[j];
}

// at[wave][d], the waves' counts, become the places of their first positions; total[d]: where the digit's first position of this
// workgroup goes.  One thread a digit.
__device__ __forceinline__ void place_waves(uint32_t (&n)[kSortWaves], uint32_t *at, int stride, int d, uint32_t place) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        at[w * stride + d] = place;
        place += n[w];
    }
}

// A lane's positions: round r of wave w takes 64 neighbours, waves follow each other.  -1: past the end.
template <int R>
__device__ __forceinline__ int sort_item(const SortParams &p, int r) {
    const long i = (long)blockIdx.x * kSortThreads * R + (threadIdx.x >> 6) * 64 * R + 64 * r + (threadIdx.x & 63);
    return i < p.M ? (int)i : -1;
}

template <int R>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortParams p, int pass) {
    if (clear_slice(p)) return;
    __shared__ uint32_t h[1 << kMaxBits];
    const int bins = 1 << p.bits;
    uint32_t key[R], digit[R], earlier[R];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = sort_item<R>(p, r) >= 0 ? sort_key(p, pass, sort_item<R>(p, r)) : 0;
    if ((int)threadIdx.x < bins) h[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        live[r] = sort_item<R>(p, r) >= 0;
        digit[r] = (key[r] >> (pass * p.bits)) & (bins - 1);
    }
    count_digits<R>(live, digit, h, p.bits, earlier);
    __syncthreads();
    if ((int)threadIdx.x < bins) p.hist[(long)blockIdx.x * bins + threadIdx.x] = h[threadIdx.x];
}

// Counts of many workgroups: each becomes the sum over the workgroups before, the whole sum goes to totals.  64 digits a
// workgroup, 16 row lanes that take a run of the counts each.
__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(const SortParams p) {
    __shared__ uint32_t part[kSortWaves][64];
    const int bins = 1 << p.bits, c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int d = blockIdx.x * 64 + c;
    const int len = (p.blocks + kSortWaves - 1) / kSortWaves, begin = min(p.blocks, r * len), end = min(p.blocks, begin + len);
    uint32_t sum = 0;
    if (d < bins)
#pragma unroll 8
        for (int b = begin; b < end; ++b) sum += p.hist[(long)b * bins + d];
    part[r][c] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        before += w < r ? part[w][c] : 0;
        all += part[w][c];
    }
    if (d < bins) {
        if (r == 0) p.totals[d] = all;
#pragma unroll 8
        for (int b = begin; b < end; ++b) {
            const uint32_t n = p.hist[(long)b * bins + d];
            p.hist[(long)b * bins + d] = before;
            before += n;
        }
    }
}

template <int R>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const SortParams p, int pass) {
    if (clear_slice(p)) return;
    __shared__ uint32_t at[kSortWaves][1 << kMaxBits];      // per wave and digit: positions, then the place of the first
    __shared__ uint32_t total[1 << kMaxBits];
    const int bins = 1 << p.bits, wave = threadIdx.x >> 6, shift = pass * p.bits;
    const int d = threadIdx.x;                               // bins <= 512: at most one digit per thread
    uint32_t key[R], digit[R], earlier[R];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = sort_item<R>(p, r) >= 0 ? sort_key(p, pass, sort_item<R>(p, r)) : 0;
    for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) at[i >> p.bits][i & (bins - 1)] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        live[r] = sort_item<R>(p, r) >= 0;
        digit[r] = (key[r] >> shift) & (bins - 1);
    }
    count_digits<R>(live, digit, at[wave], p.bits, earlier);
    uint32_t before = 0, sum = 0;
    if (p.totals && d < bins) {
        before = p.hist[(long)blockIdx.x * bins + d];
        sum = p.totals[d];
    } else if (d < bins) {
        const uint32_t *h = p.hist + d;
#pragma unroll 16
        for (int b = 0; b < p.blocks; ++b) {
            const uint32_t n = h[(long)b * bins];
            before += b < (int)blockIdx.x ? n : 0;
            sum += n;
        }
    }
    if (d < bins) total[d] = sum;
    __syncthreads();
    uint32_t n[kSortWaves] = {};
    if (d < bins)
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) n[w] = at[w][d];
    if (wave == 0) scan_totals(total, bins);
    __syncthreads();
    if (d < bins) place_waves(n, at[0], 1 << kMaxBits, d, total[d] + before);
    __syncthreads();
    uint32_t *keys_out = p.keys[pass & 1], *pos_out = p.pos[pass & 1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = sort_item<R>(p, r);
        if (i < 0) continue;
        const uint32_t place = at[wave][digit[r]] + earlier[r];
        keys_out[place] = key[r];
        pos_out[place] = pass == 0 ? (uint32_t)i : p.pos[(pass - 1) & 1][i];
    }
}

// All digits of up to 8192 positions by one workgroup: key and position of an item in one word (ids below 2^19), which
// moves through LDS from digit to digit.
constexpr int kSmallPosBits = 13, kSmallBits = 8;
template <int R>
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const SortParams p) {
    if (clear_slice(p)) return;
    __shared__ uint32_t item[kSortThreads * R];
    __shared__ uint32_t at[kSortWaves][1 << kSmallBits];
    __shared__ uint32_t total[1 << kSmallBits];
    const int bins = 1 << p.bits, wave = threadIdx.x >> 6, d = threadIdx.x;
    uint32_t v[R], digit[R], earlier[R];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = sort_item<R>(p, r);
        live[r] = i >= 0;
        v[r] = i >= 0 ? sort_key(p, 0, i) << kSmallPosBits | (uint32_t)i : 0;
    }
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = kSmallPosBits + pass * p.bits;
        for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) at[i >> p.bits][i & (bins - 1)] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) digit[r] = (v[r] >> shift) & (bins - 1);
        count_digits<R>(live, digit, at[wave], p.bits, earlier);
        __syncthreads();
        uint32_t n[kSortWaves] = {};
        if (d < bins) {
            uint32_t sum = 0;
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                n[w] = at[w][d];
                sum += n[w];
            }
            total[d] = sum;
        }
        __syncthreads();
        if (wave == 0) scan_totals(total, bins);
        __syncthreads();
        if (d < bins) place_waves(n, at[0], 1 << kSmallBits, d, total[d]);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (live[r]) item[at[wave][digit[r]] + earlier[r]] = v[r];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (live[r]) v[r] = item[sort_item<R>(p, r)];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = sort_item<R>(p, r);
        if (i < 0) continue;
        p.keys[0][i] = v[r] >> kSmallPosBits;
        p.pos[0][i] = v[r] & ((1u << kSmallPosBits) - 1);
    }
}

// ---- segmented sum ----------------------------------------------------------------------------------------
// A workgroup takes kSumWaves pieces of P positions, a span; each wave sums the runs of its piece, and where a run goes on
// into the next piece the sums are handed over in LDS.  What crosses the workgroup's ends goes to memory, one row at either
// end, for segment_join_kernel.  HBM bound: 65536 x 768 f32 rows into 10 are 31 us (181 MB, 5.8 TB/s); the sort and the join
// around it add 14.  Pieces of 32, where 4 to 16 waves and pieces of 8 and 16 are within 10 % and none faster.  Up to 8192
// positions the chip is not full and a wave's time is its piece's: pieces of 8 (sum of 5632 rows of 64: 10.4 -> 4.7 us, of
// 1024 rows of 768: 13.1 -> 5.4 us).
constexpr int kSumWaves = 8, kPiece = 32, kSmallPiece = 8;
struct SumParams {
    const uint32_t *keys, *pos;       // sorted
    const void *dy;
    long ld_dy;
    float *out;                       // [vocab, E]
    float *partial;                   // [spans][2][part_ld]: run from the span before, run into the span after
    int part_ld;
    int M, E, span, spans, accumulate;
    uint32_t vocab;
    float scale;
};

template <bool LOOSE>
__device__ __forceinline__ void write_row(const SumParams &p, uint32_t key, int col, const float (&acc)[VEC]) {
    float v[VEC];
    float *dst = p.out + (long)key * p.E + col;
    if (p.accumulate) {
        tc_load_row<float, VEC, LOOSE>(dst, v, p.E - col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] += p.scale * acc[j];
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = p.scale * acc[j];
    }
    tc_store_row<float, VEC, LOOSE>(dst, v, p.E - col);
}

template <typename T, bool LOOSE, int P>
__global__ __launch_bounds__(64 * kSumWaves) void segment_sum_kernel(const SumParams p) {
    __shared__ float rows[kSumWaves][2][VEC][64];            // [wave][run from before / run into after]
    __shared__ int open[kSumWaves];                          // bit 0: a run comes from before, 1: one goes on, 2: they are the same
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int begin = (blockIdx.x * kSumWaves + wave) * P, n = min(P, p.M - begin);      // n <= 0: nothing left
    const int col = blockIdx.y * 64 * VEC + lane * VEC;
    const bool in = col < p.E;
    int flags = 0, first_key = -1, last_key = -1;
    if (n > 0) {
        const int mine = begin + min(lane, n - 1);
        const int keys = (int)p.keys[mine], pos = (int)p.pos[mine];
        const int before = begin > 0 ? (int)p.keys[begin - 1] : -1;
        const int after = begin + n < p.M ? (int)p.keys[begin + n] : -1;
        first_key = __builtin_amdgcn_readfirstlane(keys);
        last_key = __builtin_amdgcn_readlane(keys, n - 1);
        // padding and ids out of range fill the end of the list
        const int live = __popcll(__ballot(lane < n && (uint32_t)keys != p.vocab));
        if (live > 0 && before == first_key) flags |= 1;
        if (live == n && after == last_key) flags |= 2;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        int run = 0;                                         // where the current run starts in the piece
        constexpr int U = 8;                                 // rows in flight
        for (int i0 = 0; i0 < live; i0 += U) {
            float v[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = __builtin_amdgcn_readlane(pos, min(i0 + u, live - 1));
                if (in) tc_load_row<T, VEC, LOOSE>(static_cast<const T *>(p.dy) + (long)(uint32_t)at * p.ld_dy + col, v[u], p.E - col);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i >= live) break;
                const int key = __builtin_amdgcn_readlane(keys, i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
                if (i + 1 < n && __builtin_amdgcn_readlane(keys, min(i + 1, 63)) == key) continue;
                const bool from_before = run == 0 && (flags & 1), into_after = i + 1 == n && (flags & 2);
                if (from_before || into_after) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) rows[wave][from_before ? 0 : 1][j][lane] = acc[j];
                    if (from_before && into_after) flags |= 4;
                } else if (in) {
                    write_row<LOOSE>(p, (uint32_t)key, col, acc);
                }
                run = i + 1;
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
            }
        }
    }
    if (lane == 0) open[wave] = flags;
    __syncthreads();
    // Runs that leave a piece: the wave in which such a run starts (for a run from before the workgroup: wave 0) adds the
    // parts of the waves that follow, in order.
    const bool from_before = wave == 0 && (flags & 1), starts = (flags & 2) && !(flags & 4);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 0 ? !from_before : !starts) continue;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = rows[wave][which][j][lane];
        bool goes_on = which == 1 || (flags & 4);
        for (int w = wave + 1; w < kSumWaves && goes_on; ++w) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += rows[w][0][j][lane];
            goes_on = (open[w] & 4) != 0;
        }
        if (!in) continue;
        if (which == 1 && !goes_on) write_row<LOOSE>(p, (uint32_t)last_key, col, acc);
        else tc_store_row<float, VEC>(p.partial + ((long)blockIdx.x * 2 + which) * p.part_ld + col, acc);
    }
}

// Runs over several spans: the workgroup of the span in which the run starts adds the rows, every wave kJoin of them in turn,
// and the waves' sums in order.  (One wave a run, eight rows in flight: 1048576 x 64 rows into 10 take 175 instead of 91 us.)
constexpr int kJoinWaves = 8, kJoin = 16;
template <bool LOOSE>
__global__ __launch_bounds__(64 * kJoinWaves) void segment_join_kernel(const SumParams p) {
    __shared__ float sums[kJoinWaves][VEC][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x;                                // c + 1 < spans
    const long begin = (long)c * p.span;
    const uint32_t key = p.keys[begin + p.span - 1];
    if (key == p.vocab || p.keys[begin + p.span] != key) return;
    if (begin > 0 && p.keys[begin - 1] == key) return;       // starts earlier
    const int col = blockIdx.y * 64 * VEC + lane * VEC;
    const bool in = col < p.E;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (wave == 0 && in) tc_load_row<float, VEC>(p.partial + ((long)c * 2 + 1) * p.part_ld + col, acc);
    for (long k0 = c + 1 + wave * kJoin; k0 < p.spans; k0 += kJoinWaves * kJoin) {
        // the spans that begin inside the run follow each other without a gap
        const long k = k0 + lane;
        const int n = __popcll(__ballot(lane < kJoin && k < p.spans && p.keys[min(k, (long)p.spans - 1) * p.span] == key));
        if (n == 0) break;
        float v[kJoin][VEC];
#pragma unroll
        for (int i = 0; i < kJoin; ++i)
            if (in) tc_load_row<float, VEC>(p.partial + (k0 + min(i, n - 1)) * 2 * p.part_ld + col, v[i]);
#pragma unroll
        for (int i = 0; i < kJoin; ++i)
            if (i < n)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += v[i][j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave != 0 || !in) return;
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += sums[w][j][lane];
    write_row<LOOSE>(p, key, col, acc);
}

struct BwdPlan {
    bool small;
    int rounds, blocks, passes, bits, piece, spans, part_ld;
    size_t keys[2], pos[2], hist, totals, partial, total;
};
BwdPlan bwd_plan(long M, long E, long vocab) {
    BwdPlan w{};
    if (M <= kFew) { w.total = 16; return w; }
    int bits = 0;
    while ((vocab >> bits) != 0) ++bits;           // keys 0 .. vocab
    w.small = M <= 1 << kSmallPosBits && bits + kSmallPosBits <= 32;
    const int most = w.small ? kSmallBits : kMaxBits;
    w.passes = (bits + most - 1) / most;
    w.bits = (bits + w.passes - 1) / w.passes;
    // A workgroup scatters its positions line by line, so few of them are dealt to many workgroups: up to 131072 rows 1 round each
    // (65536 rows of 64 into 50000: 38 us, with 4 rounds 49).  Up to kFewBlocks workgroups each sums the counts of the others by
    // itself, which is one launch less; with more of them that grows with the square.
    w.rounds = w.small ? (M <= 4 * kSortThreads ? 4 : 8) : M > (long)kFewBlocks * kSortThreads ? 4 : 1;
    w.blocks = (int)((M + kSortThreads * w.rounds - 1) / (kSortThreads * w.rounds));
    w.piece = M <= 8192 ? kSmallPiece : kPiece;
    w.spans = (int)((M + kSumWaves * w.piece - 1) / (kSumWaves * w.piece));
    w.part_ld = (int)((E + 3) / 4 * 4);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off += (bytes + 255) & ~(size_t)255;
        return o;
    };
    for (int k = 0; k < 2; ++k) { w.keys[k] = take((size_t)M * 4); w.pos[k] = take((size_t)M * 4); }
    w.hist = take((size_t)w.blocks * (1 << w.bits) * 4);
    w.totals = take((size_t)(1 << w.bits) * 4);
    w.partial = take((size_t)w.spans * 2 * w.part_ld * 4);
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
    // 16-byte stores, 4 f32 or 8 bf16 values; rows that start anywhere or end inside a piece take the loose form
    const int wide = out_dtype == TC_BF16 ? 8 : 4;
    const bool loose = !(tc_rows_aligned(table, E, t_esz, wide) && tc_rows_aligned(out, E, o_esz, wide));
    const int pieces = (E + wide - 1) / wide;
    int lanes_log2 = 0;
    while (lanes_log2 < 6 && (1 << lanes_log2) < pieces) ++lanes_log2;
    long blocks = ((M << lanes_log2) + 255) / 256;
    if (blocks > (1L << 20)) blocks = 1L << 20;    // a launch holds fewer than 2^32 threads; rows are walked with the grid's stride
    hipStream_t s = static_cast<hipStream_t>(stream);
    TcProfScope prof(TC_PROF_EMBED, s, (double)M * E * o_esz);
#define TC_EMB(TT, TO, TID, V, L)                                                                           \
    TC_LAUNCH((embedding_kernel<TT, TO, TID, V, L>), dim3((unsigned)blocks), dim3(256), 0, s,               \
              static_cast<const TID *>(tokens), static_cast<const TT *>(table), static_cast<TO *>(out), M, E, vocab, scale, \
              pad_idx, lanes_log2, bad)
#define TC_EMB_ID(TT, TO, V, L) do { if (id_bytes == 4) TC_EMB(TT, TO, int32_t, V, L); else TC_EMB(TT, TO, int64_t, V, L); } while (0)
#define TC_EMB_L(TT, TO, V) do { if (loose) TC_EMB_ID(TT, TO, V, true); else TC_EMB_ID(TT, TO, V, false); } while (0)
    if (table_dtype == TC_F32) {
        if (out_dtype == TC_F32) TC_EMB_L(float, float, 4);
        else TC_EMB_L(float, uint16_t, 8);
    } else {
        if (out_dtype == TC_F32) TC_EMB_L(uint16_t, float, 4);
        else TC_EMB_L(uint16_t, uint16_t, 8);
    }
#undef TC_EMB_L
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
    char *ws = static_cast<char *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool loose = !(tc_rows_aligned(dy, ld_dy, esz, VEC) && tc_rows_aligned(d_table, E, 4, VEC));
    const unsigned slabs = (unsigned)((E + 64 * VEC - 1) / (64 * VEC));
#define TC_EMB_T(KERNEL, GRID, BLOCK, P)                                                                                        \
    do {                                                                                                                        \
        if (dy_dtype == TC_F32) {                                                                                               \
            if (loose) TC_LAUNCH((KERNEL(float, true)), GRID, dim3(BLOCK), 0, s, P);                                            \
            else TC_LAUNCH((KERNEL(float, false)), GRID, dim3(BLOCK), 0, s, P);                                                 \
        } else {                                                                                                                \
            if (loose) TC_LAUNCH((KERNEL(uint16_t, true)), GRID, dim3(BLOCK), 0, s, P);                                         \
            else TC_LAUNCH((KERNEL(uint16_t, false)), GRID, dim3(BLOCK), 0, s, P);                                              \
        }                                                                                                                       \
    } while (0)
    if (M <= kFew) {
        FewParams f{};
        f.tokens = tokens; f.dy = dy; f.out = d_table; f.ld_dy = ld_dy; f.vocab = vocab; f.pad_idx = pad_idx;
        f.M = (int)M; f.E = E; f.accumulate = accumulate; f.scale = scale;
        const long want = (vocab + 3) / 4, most = 8192 / slabs > 256 ? 8192 / slabs : 256;
        const dim3 grid((unsigned)(want < most ? want : most), slabs);
#define TC_FEW4(T, L) few_positions_kernel<T, int32_t, L>
#define TC_FEW8(T, L) few_positions_kernel<T, int64_t, L>
        if (id_bytes == 4) TC_EMB_T(TC_FEW4, grid, 256, f);
        else TC_EMB_T(TC_FEW8, grid, 256, f);
        TC_CHECK_LAUNCH("tc_embedding_bwd");
        return TC_OK;
    }
    SortParams sp{};
    sp.tokens = tokens;
    sp.id_bytes = id_bytes;
    sp.M = (int)M; sp.blocks = w.blocks; sp.bits = w.bits; sp.passes = w.passes;
    sp.vocab = vocab; sp.pad_idx = pad_idx;
    sp.hist = reinterpret_cast<uint32_t *>(ws + w.hist);
    if (w.blocks > kFewBlocks) sp.totals = reinterpret_cast<uint32_t *>(ws + w.totals);
    for (int k = 0; k < 2; ++k) {
        sp.keys[k] = reinterpret_cast<uint32_t *>(ws + w.keys[k]);
        sp.pos[k] = reinterpret_cast<uint32_t *>(ws + w.pos[k]);
    }
    // the launches of the sort clear a slice of the gradient each, 64 KiB and more per workgroup
    const int launches = w.small ? 1 : 2 * w.passes;
    const long cells = accumulate ? 0 : vocab * E;
    int launch = 0;
    auto grid_of = [&]() {
        sp.clear = d_table;
        sp.clear_from = cells / 4 * launch / launches * 4;
        ++launch;
        sp.clear_to = launch == launches ? cells : cells / 4 * launch / launches * 4;
        const long wgs = (sp.clear_to - sp.clear_from + 16383) / 16384;
        return dim3((unsigned)(w.blocks + (wgs < 512 ? wgs : 512)));
    };
#define TC_SORT(KERNEL)                                                                                         \
    do {                                                                                                        \
        const dim3 grid = grid_of();                                                                            \
        if (w.rounds == 1) TC_LAUNCH(KERNEL<1>, grid, dim3(kSortThreads), 0, s, sp, pass);                      \
        else TC_LAUNCH(KERNEL<4>, grid, dim3(kSortThreads), 0, s, sp, pass);                                    \
    } while (0)
    if (w.small) {
        const dim3 grid = grid_of();
        if (w.rounds == 4) TC_LAUNCH(sort_small_kernel<4>, grid, dim3(kSortThreads), 0, s, sp);
        else TC_LAUNCH(sort_small_kernel<8>, grid, dim3(kSortThreads), 0, s, sp);
    } else {
        for (int pass = 0; pass < w.passes; ++pass) {
            TC_SORT(sort_count_kernel);
            if (sp.totals) TC_LAUNCH(sort_scan_kernel, dim3((unsigned)(((1 << w.bits) + 63) / 64)), dim3(kSortThreads), 0, s, sp);
            TC_SORT(sort_place_kernel);
        }
    }
#undef TC_SORT
    SumParams q{};
    const int sorted = w.small ? 0 : (w.passes - 1) & 1;
    q.keys = sp.keys[sorted]; q.pos = sp.pos[sorted];
    q.dy = dy; q.ld_dy = ld_dy;
    q.out = d_table;
    q.partial = reinterpret_cast<float *>(ws + w.partial);
    q.part_ld = w.part_ld;
    q.M = (int)M; q.E = E; q.span = kSumWaves * w.piece; q.spans = w.spans;
    q.accumulate = accumulate; q.vocab = (uint32_t)vocab; q.scale = scale;
#define TC_SUM(T, L) segment_sum_kernel<T, L, kPiece>
#define TC_SUM_SMALL(T, L) segment_sum_kernel<T, L, kSmallPiece>
    if (w.piece == kPiece) TC_EMB_T(TC_SUM, dim3((unsigned)w.spans, slabs), 64 * kSumWaves, q);
    else TC_EMB_T(TC_SUM_SMALL, dim3((unsigned)w.spans, slabs), 64 * kSumWaves, q);
    if (w.spans > 1) {
        if (loose) TC_LAUNCH(segment_join_kernel<true>, dim3((unsigned)w.spans - 1, slabs), dim3(64 * kJoinWaves), 0, s, q);
        else TC_LAUNCH(segment_join_kernel<false>, dim3((unsigned)w.spans - 1, slabs), dim3(64 * kJoinWaves), 0, s, q);
    }
#undef TC_SUM_SMALL
#undef TC_SUM
#undef TC_FEW8
#undef TC_FEW4
#undef TC_EMB_T
    TC_CHECK_LAUNCH("tc_embedding_bwd");
    return TC_OK;
}
