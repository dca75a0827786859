// Table lookup out[i] = scale * W[ids[i]] and its gradient dW[v] = scale * sum over ids[i] == v of g[i].
//
// The gradient of a table of a few rows sums into tables in LDS, one for every group of lanes that walks over rows.  That of
// a larger one sorts the token ids (stable radix sort on (id, position) pairs) and sums the rows of g in sorted order: the
// occurrences of one token become one RUN of neighbouring slots.  Slots are cut into tiles of equal length, so the reading of g
// is even however often a token occurs; a run inside one tile is finished there, a run over several tiles leaves one fp32
// partial row per tile and a second launch joins them, a workgroup for each run and 256 columns (slow for a run of very many).  No floating-point atomics: the order of every sum depends on the
// sizes and the ids alone.
#include "common.h"

namespace {

constexpr int64_t kMaxWidth = 1 << 15;                   // (1024 + pieces) * pieces < 2^32 for the division in the forward
constexpr int64_t kMaxPieces = (int64_t)1 << 33;         // work-items of a launch stay below 2^32

template <bool I64>
__device__ __forceinline__ int64_t ld_id(const void* __restrict__ ids, int64_t i) {
    return I64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// A row is moved in pieces of W elements, 16 bytes, at whatever alignment it has (the hardware takes any; the compiler is
// promised the element's).  The last piece of a row whose width is no multiple of W begins W before the row's end: its first
// elements are the piece before's once more, with the same values.  NARROW: rows of less than W elements, one by one.
template <class T>
struct alignas(16) Piece {
    static constexpr int W = 16 / sizeof(T);
    T v[W];
};
template <class T, bool NARROW>
__device__ __forceinline__ int piece_column(int q, int D) {
    const int c = q * Piece<T>::W;
    return NARROW ? 0 : c < D - Piece<T>::W ? c : D - Piece<T>::W;
}
template <class T, bool NARROW>
__device__ __forceinline__ void ld_piece(Piece<T>& x, const T* __restrict__ p, int D) {
    if (NARROW) {
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) x.v[k] = k < D ? p[k] : (T)0.f;
    } else __builtin_memcpy(&x, p, 16);
}
template <class T, bool NARROW>
__device__ __forceinline__ void st_piece(T* __restrict__ p, int D, const Piece<T>& x) {
    if (NARROW) {
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) if (k < D) p[k] = x.v[k];
    } else __builtin_memcpy(p, &x, 16);
}
template <class T, bool NARROW>
__device__ __forceinline__ void st_scaled(T* __restrict__ p, int D, const float (&acc)[Piece<T>::W], float scale) {
    Piece<T> x;
#pragma unroll
    for (int k = 0; k < Piece<T>::W; ++k) x.v[k] = (T)(acc[k] * scale);
    st_piece<T, NARROW>(p, D, x);
}
template <class T, bool NARROW>
__device__ __forceinline__ void st_sums(float* __restrict__ p, int D, const float (&acc)[Piece<T>::W]) {
    if (NARROW) {
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) if (k < D) p[k] = acc[k];
    } else __builtin_memcpy(p, acc, sizeof(acc));
}

// ------------------------------------------------------------------------------------------------ forward
// The output is a flat row of n * nv pieces; a thread moves U pieces 256 apart, so stores are contiguous whatever the width.
// Piece -> row needs a division by nv: the block's first row comes from one 64-bit division (scalar), the rest from a
// multiplication by `magic` = ceil(2^32 / nv), exact while (256 U + nv) * nv < 2^32.
// Bound by the bytes written (and read, where the table is larger than the caches): 1,048,576 x 128 fp32 from 7 rows 99 us
// (5.4 TB/s), 65,537 x 520 fp16 from 131,071 rows 31 us (4.4 TB/s read and written, rows at any alignment), 16,384 x 1,024
// bf16 10.8 us (33.6 MB: a launch's own 2.5 us count).
template <class T, int U, bool I64, bool NARROW, bool STREAM>      // STREAM: an output that no cache holds
__global__ __launch_bounds__(256) void k_embedding_fwd(const T* __restrict__ w, int64_t ldw, int64_t V, const void* __restrict__ ids,
                                                       int64_t n, uint32_t nv, uint32_t magic, int D, float scale, T* __restrict__ out,
                                                       int64_t ldo) {
    const int64_t total = n * nv, p0 = (int64_t)blockIdx.x * (256 * U);
    const int64_t row0 = p0 / nv;
    const uint32_t rem0 = (uint32_t)(p0 - row0 * nv);
    int64_t row[U], id[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t o = rem0 + threadIdx.x + 256 * u;
        const uint32_t q = magic ? __umulhi(o, magic) : o;                 // magic 0: nv == 1
        row[u] = row0 + q;
        col[u] = piece_column<T, NARROW>((int)(o - q * nv), D);
        id[u] = p0 + threadIdx.x + 256 * u < total ? ld_id<I64>(ids, row[u]) : -1;
    }
    Piece<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (id[u] >= 0 && id[u] < V) ld_piece<T, NARROW>(x[u], w + id[u] * ldw + col[u], D);
        else
#pragma unroll
            for (int k = 0; k < Piece<T>::W; ++k) x[u].v[k] = (T)0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (p0 + threadIdx.x + 256 * u >= total) continue;
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) x[u].v[k] = (T)((float)x[u].v[k] * scale);
        T* p = out + row[u] * ldo + col[u];
        if (STREAM) {
            typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
            Words v;
            __builtin_memcpy(&v, &x[u], 16);
            __builtin_nontemporal_store(v, reinterpret_cast<Words*>(p));
        } else st_piece<T, NARROW>(p, D, x[u]);
    }
}

// ------------------------------------------------------------------------------------------------ gradient of a few rows
// LG lanes walk over rows of g, four elements each (8 or 16 bytes; the last lane's begin four before the row's end); their
// sums of every table row stand in LDS, a float4 for every table row and lane that no other lane touches.  The block's
// groups are added up in order and leave one partial table, the blocks' tables are added up by a second launch.
// g is read once and nothing else is large: 1,048,576 x 128 fp32 into 7 rows 94 us + 7 us for the blocks' tables (537 MB,
// 5.3 TB/s).  LDS is what limits it: a row more is 4 KB a block, so with more rows fewer loads are in flight (20 rows 46 us
// against 56 us sorted at 262,144 x 128 fp32, 32 rows 93 us against 54 us: the sort from 21 rows on).
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; };
template <class T, bool I64, bool NARROW>      // NARROW: D < 4
__global__ __launch_bounds__(256) void k_embedding_few(const void* __restrict__ ids, int64_t n, int V, const T* __restrict__ g, int64_t ldg,
                                                       int D, float* __restrict__ part, int LG, int64_t chunk) {
    constexpr int U = sizeof(T) == 4 ? 4 : 8;            // 64 bytes in flight a lane
    extern __shared__ float4 table[];                    // [V][256]
    const int t = threadIdx.x, lane = t & (LG - 1), group = t / LG, groups = 256 / LG, q = blockIdx.y * LG + lane;
    const int col = NARROW ? 0 : 4 * q < D - 4 ? 4 * q : D - 4;
    const bool here = 4 * q < D;
    for (int v = 0; v < V; ++v) table[v * 256 + t] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int64_t r0 = blockIdx.x * chunk, r1 = r0 + chunk < n ? r0 + chunk : n;
    if (here)
        for (int64_t r = r0 + group; r < r1; r += groups * U) {
            int64_t id[U];
            Four<T> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) id[u] = r + u * groups < r1 ? ld_id<I64>(ids, r + u * groups) : -1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (id[u] < 0 || id[u] >= V) continue;
                const T* p = g + (r + u * groups) * ldg + col;
                if (!NARROW) x[u] = *reinterpret_cast<const Four<T>*>(p);
                else
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[u].v[k] = k < D ? p[k] : (T)0.f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (id[u] < 0 || id[u] >= V) continue;
                float4& s = table[(int)id[u] * 256 + t];
                s = bg_add4(s, make_float4((float)x[u].v[0], (float)x[u].v[1], (float)x[u].v[2], (float)x[u].v[3]));
            }
        }
    __syncthreads();
    if (group == 0 && here)
        for (int v = 0; v < V; ++v) {
            float4 s = table[v * 256 + lane];
            for (int y = 1; y < groups; ++y) s = bg_add4(s, table[v * 256 + y * LG + lane]);
            float* p = part + ((int64_t)blockIdx.x * V + v) * D + col;
            p[0] = s.x;
            if (!NARROW || D > 1) p[1] = s.y;
            if (!NARROW || D > 2) p[2] = s.z;
            if (!NARROW) p[3] = s.w;
        }
}

constexpr int kFewCols = 32, kFewSplit = 8;
template <class T>
__global__ __launch_bounds__(kFewCols* kFewSplit) void k_embedding_few_join(const float* __restrict__ part, int64_t blocks, int64_t size,
                                                                            float scale, T* __restrict__ dw) {
    __shared__ float sum[kFewSplit][kFewCols];
    const int tx = threadIdx.x % kFewCols, ty = threadIdx.x / kFewCols;
    const int64_t c = (int64_t)blockIdx.x * kFewCols + tx;
    float s = 0.f;
    if (c < size)
#pragma unroll 8
        for (int64_t b = ty; b < blocks; b += kFewSplit) s += part[b * size + c];
    sum[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < size) {
        for (int y = 1; y < kFewSplit; ++y) s += sum[y][tx];
        dw[c] = (T)(s * scale);
    }
}

// ------------------------------------------------------------------------------------------------ stable sort of the ids
// Least significant digit first, one pass = a histogram per tile of keys and a placement.  The key of a missing token is
// V, behind every row.  Both launches carry extra workgroups that zero a share of dW meanwhile: the sort of a batch's
// tokens is bound by latency, not by memory (16,384 tokens of 32,000: four launches, 25 us, which the 65 MB of zeros fit
// into; 65,537 of 131,071: 41 us and 136 MB).
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;
constexpr int kSortThreads = 512;

struct Fill { uint4* p; int64_t n16; };                  // n16 pieces of 16 bytes

__device__ __forceinline__ void d_fill(Fill f, int64_t block, int64_t blocks) {
    for (int64_t i = block * kSortThreads + threadIdx.x; i < f.n16; i += blocks * kSortThreads) f.p[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <int SRC>      // 0: int64 ids, 1: int32 ids, 2: keys of an earlier pass
__device__ __forceinline__ int32_t ld_key(const void* __restrict__ src, int64_t i, int64_t V) {
    if (SRC == 2) return static_cast<const int32_t*>(src)[i];
    const int64_t id = ld_id<SRC == 0>(src, i);
    return (int32_t)(id >= 0 && id < V ? id : V);
}

// hist[tile][bin], or [bin][tile] where a scan over the tiles follows
template <int SRC, int ROUNDS>
__global__ __launch_bounds__(kSortThreads) void k_sort_hist(const void* __restrict__ src, int64_t n, int64_t V, int shift, int bins,
                                                            int32_t* __restrict__ hist, int n_tiles, bool scanned, Fill fill) {
    if ((int)blockIdx.x >= n_tiles) { d_fill(fill, blockIdx.x - n_tiles, gridDim.x - n_tiles); return; }
    __shared__ int32_t h[kBins];
    if (threadIdx.x < kBins) h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (kSortThreads * ROUNDS);
    int32_t key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = base + r * kSortThreads + threadIdx.x;
        key[r] = i < n ? ld_key<SRC>(src, i, V) : -1;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (key[r] >= 0) atomicAdd(&h[(key[r] >> shift) & (bins - 1)], 1);
    __syncthreads();
    if ((int)threadIdx.x < bins)
        hist[scanned ? (int64_t)threadIdx.x * n_tiles + blockIdx.x : (int64_t)blockIdx.x * bins + threadIdx.x] = h[threadIdx.x];
}

// in place: hist[bin][tile] -> number of that bin's keys in earlier tiles; total[bin] = all of them.  One wave per bin.
__global__ __launch_bounds__(256) void k_sort_scan(int32_t* __restrict__ hist, int n_tiles, int bins, int32_t* __restrict__ total) {
    const int bin = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (bin >= bins) return;
    int32_t* h = hist + (int64_t)bin * n_tiles;
    int32_t carry = 0;
    for (int t0 = 0; t0 < n_tiles; t0 += 64) {
        const int t = t0 + lane;
        const int32_t v = t < n_tiles ? h[t] : 0;
        int32_t x = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int32_t y = __shfl_up(x, off, 64);
            if (lane >= off) x += y;
        }
        if (t < n_tiles) h[t] = carry + x - v;
        carry += __shfl(x, 63, 64);
    }
    if (lane == 0) total[bin] = carry;
}

// Rank of this lane's digit among the wave's equal digits of earlier rounds and lower lanes; counts them in cnt (the wave's own
// row: LDS keeps a wave's accesses in order).  Ballots over the digit's bits find the lanes that have the same one.
template <class Count>
__device__ __forceinline__ int wave_rank(int d, bool valid, int bits, Count* cnt) {
    const uint64_t live = __ballot(valid);
    uint32_t lo = (uint32_t)live, hi = (uint32_t)(live >> 32);
    for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((d >> b) & 1);
        const uint32_t same = 0u - ((d >> b) & 1);       // lanes whose bit is this lane's: ~(m ^ same)
        lo &= ~((uint32_t)m ^ same);
        hi &= ~((uint32_t)(m >> 32) ^ same);
    }
    const int below = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0)), c = cnt[d];
    __builtin_amdgcn_wave_barrier();
    if (valid && below == 0) cnt[d] = (Count)(c + __popc(lo) + __popc(hi));
    __builtin_amdgcn_wave_barrier();
    return c + below;
}

// All passes of up to kSmall keys by one workgroup, keys and positions in registers and LDS; the other workgroups zero dW.
// (One launch instead of two for every digit; four keys a thread measured as well as eight and sixteen.)
constexpr int kSmallThreads = 1024, kSmallRounds = 4, kSmall = kSmallThreads * kSmallRounds;
template <int SRC>
__global__ __launch_bounds__(kSmallThreads) void k_sort_small(const void* __restrict__ src, int n, int64_t V, int passes, int bits,
                                                              int32_t* __restrict__ key_out, int32_t* __restrict__ pos_out, Fill fill) {
    if (blockIdx.x > 0) {
        for (int64_t i = (int64_t)(blockIdx.x - 1) * kSmallThreads + threadIdx.x; i < fill.n16; i += (int64_t)(gridDim.x - 1) * kSmallThreads)
            fill.p[i] = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    constexpr int kWaves = kSmallThreads / 64;
    __shared__ uint64_t pairs[kSmall];                   // (key, position) in the order of the last pass
    __shared__ uint16_t cnt[kWaves][kBins];
    __shared__ int32_t wsum[kBins / 64], base[kBins];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, bins = 1 << bits;
    const int rounds = (n + kSmallThreads - 1) / kSmallThreads, first = wave * (64 * rounds) + lane;
    int32_t key[kSmallRounds], pos[kSmallRounds];
    int rank[kSmallRounds];
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const int i = first + 64 * r;
        key[r] = r < rounds && i < n ? ld_key<SRC>(src, i, V) : -1;
        pos[r] = i;
    }
    for (int q = 0; q < passes; ++q) {
        const int shift = q * bits;
        for (int i = t; i < kWaves * kBins / 2; i += kSmallThreads) reinterpret_cast<uint32_t*>(&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r)
            if (r < rounds) rank[r] = wave_rank((key[r] >> shift) & (bins - 1), key[r] >= 0, bits, cnt[wave]);
        __syncthreads();
        int32_t all = 0, x = 0;                          // exclusive sums: over the waves, then over the bins
        if (t < kBins) {
            for (int w = 0; w < kWaves; ++w) { const int32_t c = cnt[w][t]; cnt[w][t] = (uint16_t)all; all += c; }
            x = all;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int32_t y = __shfl_up(x, off, 64);
                if (lane >= off) x += y;
            }
            if (lane == 63) wsum[wave] = x;
        }
        __syncthreads();
        if (t < kBins) {
            int32_t b = x - all;
            for (int w = 0; w < wave; ++w) b += wsum[w];
            base[t] = b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r) {
            if (r >= rounds || key[r] < 0) continue;
            const int d = (key[r] >> shift) & (bins - 1), dst = base[d] + cnt[wave][d] + rank[r];
            pairs[dst] = ((uint64_t)(uint32_t)pos[r] << 32) | (uint32_t)key[r];
        }
        __syncthreads();
        if (q < passes - 1)
#pragma unroll
            for (int r = 0; r < kSmallRounds; ++r) {
                const int i = first + 64 * r;
                if (r < rounds && i < n) { const uint64_t v = pairs[i]; key[r] = (int32_t)v; pos[r] = (int32_t)(v >> 32); }
            }
    }
    for (int i = t; i < n; i += kSmallThreads) {         // (from LDS: written where they fall, every word would be a line)
        const uint64_t v = pairs[i];
        key_out[i] = (int32_t)v;
        pos_out[i] = (int32_t)(v >> 32);
    }
}

// Placement.  A wave owns 64 * ROUNDS consecutive keys; to a key's rank in its wave the waves' and the tiles' counts are
// added: stable by construction.
template <int SRC, int ROUNDS, bool SCANNED>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(const void* __restrict__ src, const int32_t* __restrict__ pos_in, int64_t n,
                                                             int64_t V, int shift, int bits, const int32_t* __restrict__ hist,
                                                             const int32_t* __restrict__ total, int n_tiles,
                                                             int32_t* __restrict__ key_out, int32_t* __restrict__ pos_out, Fill fill) {
    if ((int)blockIdx.x >= n_tiles) { d_fill(fill, blockIdx.x - n_tiles, gridDim.x - n_tiles); return; }
    constexpr int kWaves = kSortThreads / 64;
    __shared__ int32_t cnt[kWaves][kBins];
    __shared__ int32_t wsum[kWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, bins = 1 << bits;
    const int64_t first = (int64_t)blockIdx.x * (kSortThreads * ROUNDS) + wave * (64 * ROUNDS) + lane;
    int32_t key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = first + 64 * r;
        key[r] = i < n ? ld_key<SRC>(src, i, V) : -1;
        pos[r] = i < n ? (SRC == 2 ? pos_in[i] : (int32_t)i) : 0;
    }
    for (int w = 0; w < kWaves; ++w) cnt[w][t] = 0;                      // kSortThreads == kBins
    int32_t before = 0, all = 0;                                         // of bin t: keys in earlier tiles, in all tiles
    if (t < bins) {
        if (SCANNED) { before = hist[(int64_t)t * n_tiles + blockIdx.x]; all = total[t]; }
        else
#pragma unroll 8
            for (int k = 0; k < n_tiles; ++k) {
                const int32_t v = hist[(int64_t)k * bins + t];
                all += v;
                before += k < (int)blockIdx.x ? v : 0;
            }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) rank[r] = wave_rank((key[r] >> shift) & (bins - 1), key[r] >= 0, bits, cnt[wave]);
    // exclusive sum of `all` over the bins
    int32_t x = all;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int32_t base = before + x - all;
    for (int w = 0; w < wave; ++w) base += wsum[w];
    for (int w = 0; w < kWaves; ++w) { const int32_t c = cnt[w][t]; cnt[w][t] = base; base += c; }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (key[r] < 0) continue;
        const int32_t dst = cnt[wave][(key[r] >> shift) & (bins - 1)] + rank[r];
        key_out[dst] = key[r];
        pos_out[dst] = pos[r];
    }
}

// ------------------------------------------------------------------------------------------------ sums over the runs
// LG lanes carry one tile of C slots over LG pieces of a row.  They read LG slots at a time, one each, and pass them round.
// part[(2 * tile + which) * D + c]: which 0 = the run that began in an earlier tile, 1 = one that goes on into the next
// Bound by the gather of g's rows: eight loads in flight a lane, asked for whether or not the slot's token exists (35.8 ->
// 28.2 us at 65,537 x 520 fp16).  16,384 x 1,024 bf16: 10.9 us (33.6 MB read, 14.6 MB written: 4.4 TB/s).
// (a scalar where the wave carries one tile)
__device__ __forceinline__ int32_t pass_round(int32_t v, int lane, int LG) {
    return LG == 64 ? __builtin_amdgcn_readlane(v, lane) : __shfl(v, lane, LG);
}
template <class T, bool NARROW, int WIDTH>      // WIDTH 64: LG is 64, known to the compiler
__global__ __launch_bounds__(256) void k_embedding_runs(const int32_t* __restrict__ key, const int32_t* __restrict__ pos, int64_t n,
                                                        int32_t V, const T* __restrict__ g, int64_t ldg, int D, float scale,
                                                        T* __restrict__ dw, float* __restrict__ part, int C, int lanes) {
    constexpr int W = Piece<T>::W, U = 8;
    const int LG = WIDTH ? WIDTH : lanes;
    const int lane = threadIdx.x & (LG - 1);
    const int64_t tile = (int64_t)blockIdx.x * (256 / LG) + threadIdx.x / LG;
    const int q = blockIdx.y * LG + lane;
    const bool here = q < (D + W - 1) / W;
    const int col = piece_column<T, NARROW>(q, D);
    const int64_t k0 = tile * C < n ? tile * C : n, k1 = k0 + C < n ? k0 + C : n;          // (no slots behind the last tile)
    int32_t cur = k0 < k1 ? key[k0] : V;
    if (WIDTH) cur = __builtin_amdgcn_readfirstlane(cur);
    bool earlier = k0 > 0 && k0 < k1 && key[k0 - 1] == cur;
    const int32_t after = k1 < n ? key[k1] : -1;
    float acc[W];
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] = 0.f;
    for (int64_t b = k0; b < k0 + C; b += LG) {                          // the wave's groups make the same number of rounds
        const bool in = b + lane < k1;
        const int32_t my_key = in ? key[b + lane] : V, my_pos = in ? pos[b + lane] : 0;
        const int m = C < LG ? C : LG;
        for (int j = 0; j < m; j += U) {
            int32_t kk[U];
            Piece<T> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                kk[u] = pass_round(my_key, j + u, LG);
                const int32_t p = pass_round(my_pos, j + u, LG);
                ld_piece<T, NARROW>(x[u], g + (int64_t)p * ldg + col, D);       // (also where it is not wanted: no branch)
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (kk[u] != cur) {
                    if (cur < V && here) {
                        if (earlier) st_sums<T, NARROW>(part + 2 * tile * D + col, D, acc);
                        else st_scaled<T, NARROW>(dw + (int64_t)cur * D + col, D, acc, scale);
                    }
                    cur = kk[u];
                    earlier = false;
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[e] = 0.f;
                }
                if (cur < V)
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[e] += (float)x[u].v[e];
            }
        }
    }
    if (cur < V && here) {
        if (earlier) st_sums<T, NARROW>(part + 2 * tile * D + col, D, acc);
        else if (after == cur) st_sums<T, NARROW>(part + (2 * tile + 1) * D + col, D, acc);
        else st_scaled<T, NARROW>(dw + (int64_t)cur * D + col, D, acc, scale);
    }
}

// The run that begins in tile blockIdx.x and goes on: its own partial and the following tiles' are added by kJoin threads a
// column (strided over the tiles), those kJoin sums then in order.  Latency: the search for a long run's end and the walk
// over its tiles (7.6 us where a fifteenth of 16,384 tokens are one, some 70 tiles; two threads a column measured best of 2, 4,
// 8, 16 there).  The walk grows with the longest run: 1,048,576 x 64 fp32 of 100 rows 11 us with even ones, 79 us where a
// fifth of the tokens are one (1,638 tiles), 350 us where all are (8,192), beside 42 to 52 us for the sums themselves.
constexpr int kJoin = 2, kJoinCols = 64;
template <class T>
__global__ __launch_bounds__(kJoin* kJoinCols) void k_embedding_join(const int32_t* __restrict__ key, int64_t n, int32_t V,
                                                                     const float* __restrict__ part, int C, int64_t D, float scale,
                                                                     T* __restrict__ dw) {
    constexpr int E = 4;                                                 // columns per thread, kJoinCols apart
    const int64_t tile = blockIdx.x, k0 = tile * C, k1 = k0 + C;
    if (k1 >= n) return;
    const int32_t cur = key[k1 - 1], next = key[k1], head = key[k0], prev = k0 > 0 ? key[k0 - 1] : -1;
    if (cur >= V || next != cur) return;
    if (head == cur && prev == cur) return;                              // it began earlier: that tile joins it
    int64_t lo = k1 + 1, hi = n;                                         // the run's end: sought by all threads at once
    while (lo < hi) {
        const int64_t step = (hi - lo + blockDim.x - 1) / blockDim.x, k = lo + threadIdx.x * step;
        const int c = __syncthreads_count(k < hi && key[k] == cur);
        const int64_t nlo = c ? lo + (c - 1) * step + 1 : lo, nhi = c ? lo + c * step : lo;
        lo = nlo;
        hi = nhi < hi ? nhi : hi;
    }
    const int64_t last = (lo - 1) / C;                                   // the tile of its last slot
    __shared__ float sum[kJoin][E][kJoinCols];
    const int tx = threadIdx.x % kJoinCols, ty = threadIdx.x / kJoinCols;
    const int64_t c0 = (int64_t)blockIdx.y * (kJoinCols * E) + tx;
    float s[E];
    int64_t col[E];                                                      // (columns behind the last: the last once more, not stored)
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int64_t c = c0 + e * kJoinCols;
        col[e] = c < D ? c : D - 1;
        s[e] = ty == 0 ? part[(2 * tile + 1) * D + col[e]] : 0.f;
    }
    const float* rows = part + (tile + 1 + ty) * 2 * D;
    int64_t left = last - tile - ty;                                     // tiles of this thread: left / kJoin, rounded up
#pragma unroll 4
    for (; left > 0; left -= kJoin, rows += 2 * kJoin * D)
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += rows[col[e]];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[ty][e][tx] = s[e];
    __syncthreads();
    if (ty == 0)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t c = c0 + e * kJoinCols;
            for (int y = 1; y < kJoin; ++y) s[e] += sum[y][e][tx];
            if (c < D) dw[(int64_t)cur * D + c] = (T)(s[e] * scale);
        }
}

// ------------------------------------------------------------------------------------------------ host side
// Lanes a row: the most that leave little of a wave idle behind the row's last piece
int lanes_per_row(int64_t pieces) {
    int best = 8;
    for (int lg = 16; lg <= 64; lg *= 2)
        if ((pieces + lg - 1) / lg * lg * 4 <= (pieces + 7) / 8 * 8 * 5) best = lg;
    return best;
}

constexpr int64_t kFewRows = 20;       // table rows up to which the sums stand in LDS: 80 KB, two workgroups a compute unit

struct BwdPlan {                       // pieces of the workspace (bytes) and the shape of the launches: functions of n, V, D only
    bool few;
    int passes, bits, rounds, n_tiles, LG, C;
    int64_t key_a, key_b, pos_a, pos_b, hist, total, part, bytes, run_tiles, chunk, blocks;
};

BwdPlan bwd_plan(int64_t n, int64_t V, int64_t D, int elem) {
    BwdPlan p = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    p.few = V <= kFewRows;
    const int W = p.few ? 4 : 16 / elem;
    const int64_t pieces = (D + W - 1) / W;
    // in the runs a whole wave for a row from 33 pieces on, though many of its lanes may be idle behind the last one: a row's
    // lines are asked for together (65 pieces: 71 us with 64 lanes, 82 us with 16)
    p.LG = !p.few && pieces > 32 ? 64 : lanes_per_row(pieces);
    const int64_t column_blocks = (pieces + p.LG - 1) / p.LG;
    if (p.few) {
        const int64_t step = 256 / p.LG * (elem == 4 ? 4 : 8);       // rows a block takes at once
        int64_t most = 1024 / column_blocks;
        if (most < 1) most = 1;
        p.blocks = (n + 4 * step - 1) / (4 * step);
        if (p.blocks > most) p.blocks = most;
        p.chunk = ((n + p.blocks - 1) / p.blocks + step - 1) / step * step;
        p.blocks = (n + p.chunk - 1) / p.chunk;
        p.part = take(4 * p.blocks * V * D);
        p.bytes = at;
        return p;
    }
    int b = 1;
    while (V >> b) ++b;                                  // keys go up to V
    p.passes = (b + kDigitBits - 1) / kDigitBits;
    p.bits = (b + p.passes - 1) / p.passes;
    p.rounds = n <= 65536 ? 2 : n <= 131072 ? 4 : 8;     // up to 64 tiles, whose counts every workgroup adds up by itself
    p.n_tiles = (int)((n + kSortThreads * p.rounds - 1) / (kSortThreads * p.rounds));
    p.C = 128;
    while (p.C > 16 && n * column_blocks * p.LG / ((int64_t)p.C * 64) < 2048) p.C /= 2;
    p.run_tiles = (n + p.C - 1) / p.C;
    p.key_a = take(4 * n); p.key_b = take(4 * n); p.pos_a = take(4 * n); p.pos_b = take(4 * n);
    p.hist = take((int64_t)4 * kBins * p.n_tiles);
    p.total = take(4 * kBins);
    p.part = take(8 * p.run_tiles * D);
    p.bytes = at;
    return p;
}

template <class T, bool I64>
int launch_fwd(const T* w, int64_t ldw, int64_t V, const void* ids, int64_t n, int64_t D, float scale, T* out, int64_t ldo, hipStream_t s) {
    const uint32_t nv = (uint32_t)((D + Piece<T>::W - 1) / Piece<T>::W);
    const uint32_t magic = nv == 1 ? 0u : (uint32_t)(((1ull << 32) + nv - 1) / nv);
    if (n > kMaxPieces / nv) return BG_ERR_SHAPE;
    const int64_t total = n * nv;
    // an output past the last-level cache is stored around the caches (537 MB: 99 us against 125 us; 33 MB: no difference,
    // and whoever reads it next may find it there)
    const bool small = total <= 1 << 16, narrow = D < Piece<T>::W, stream = !narrow && total * 16 > ((int64_t)256 << 20);
    const auto kernel = narrow ? (small ? k_embedding_fwd<T, 1, I64, true, false> : k_embedding_fwd<T, 4, I64, true, false>)
                      : small ? k_embedding_fwd<T, 1, I64, false, false>
                      : stream ? k_embedding_fwd<T, 4, I64, false, true> : k_embedding_fwd<T, 4, I64, false, false>;
    kernel<<<bg_grid_for(total, small ? 256 : 1024, 1 << 30), 256, 0, s>>>(w, ldw, V, ids, n, nv, magic, (int)D, scale, out, ldo);
    BG_LAUNCH_CHECK();
    return BG_OK;
}

template <int SRC>
void launch_sort_pass(const BwdPlan& p, const void* src, const int32_t* pos_in, int64_t n, int64_t V, int shift, int32_t* hist,
                      int32_t* total, int32_t* key_out, int32_t* pos_out, Fill f0, Fill f1, hipStream_t s) {
    const int bins = 1 << p.bits;
    const int b0 = f0.n16 ? bg_grid_for(f0.n16, kSortThreads * 4, 1024) : 0, b1 = f1.n16 ? bg_grid_for(f1.n16, kSortThreads * 4, 1024) : 0;
    const bool scanned = p.n_tiles > 64;
    const auto hist_kernel = p.rounds == 2 ? k_sort_hist<SRC, 2> : p.rounds == 4 ? k_sort_hist<SRC, 4> : k_sort_hist<SRC, 8>;
    hist_kernel<<<p.n_tiles + b0, kSortThreads, 0, s>>>(src, n, V, shift, bins, hist, p.n_tiles, scanned, f0);
    if (scanned) k_sort_scan<<<(bins + 3) / 4, 256, 0, s>>>(hist, p.n_tiles, bins, total);
    const auto place_kernel = p.rounds == 2 ? k_sort_place<SRC, 2, false> : p.rounds == 4 ? k_sort_place<SRC, 4, false>
                            : scanned ? k_sort_place<SRC, 8, true> : k_sort_place<SRC, 8, false>;
    place_kernel<<<p.n_tiles + b1, kSortThreads, 0, s>>>(src, pos_in, n, V, shift, p.bits, hist, total, p.n_tiles, key_out, pos_out, f1);
}

template <int SRC>
int launch_sort_small(const BwdPlan& p, const void* src, int64_t n, int64_t V, int32_t* key_out, int32_t* pos_out, Fill f, hipStream_t s) {
    k_sort_small<SRC><<<1 + (f.n16 ? bg_grid_for(f.n16, kSmallThreads * 4, 1024) : 0), kSmallThreads, 0, s>>>(src, (int)n, V, p.passes,
                                                                                                               p.bits, key_out, pos_out, f);
    BG_LAUNCH_CHECK();
    return BG_OK;
}

template <class T, bool I64>
int launch_few(const BwdPlan& p, const void* ids, int64_t n, int64_t V, const T* g, int64_t ldg, int64_t D, float scale, T* dw, float* part,
               hipStream_t s) {
    const size_t lds = (size_t)V * 4096;
    const auto kernel = D < 4 ? k_embedding_few<T, I64, true> : k_embedding_few<T, I64, false>;
    if (lds > 64 * 1024) BG_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<dim3((unsigned)p.blocks, (unsigned)(((D + 3) / 4 + p.LG - 1) / p.LG)), 256, lds, s>>>(
        ids, n, (int)V, g, ldg, (int)D, part, p.LG, p.chunk);
    BG_LAUNCH_CHECK();
    k_embedding_few_join<T><<<bg_grid_for(V * D, kFewCols), kFewCols * kFewSplit, 0, s>>>(part, p.blocks, V * D, scale, dw);
    BG_LAUNCH_CHECK();
    return BG_OK;
}

__global__ void k_fill_tail(uint8_t* p, int n) { if ((int)threadIdx.x < n) p[threadIdx.x] = 0; }

bool bwd_sizes_ok(int64_t n, int64_t V, int64_t D) { return n <= ((int64_t)1 << 30) && V < ((int64_t)1 << 31) - 1 && D <= kMaxWidth; }

}  // namespace

extern "C" int bg_embedding_fwd(int dtype, const void* weight, int64_t ldw, int64_t V, const void* ids, int ids_is_64, int64_t n,
                                int64_t D, float scale, void* out, int64_t ldo, bgStream stream) {
    if (!bg_elem_size(dtype) || n < 0 || D < 0 || V < 0 || ldw < D || ldo < D) return BG_ERR_ARG;
    if (n == 0 || D == 0) return BG_OK;
    if ((V > 0 && !weight) || !ids || !out) return BG_ERR_ARG;
    if (D > kMaxWidth) return BG_ERR_SHAPE;
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T* w = static_cast<const T*>(weight);
        T* o = static_cast<T*>(out);
        hipStream_t s = (hipStream_t)stream;
        return ids_is_64 ? launch_fwd<T, true>(w, ldw, V, ids, n, D, scale, o, ldo, s) : launch_fwd<T, false>(w, ldw, V, ids, n, D, scale, o, ldo, s);
    });
}

extern "C" int64_t bg_embedding_bwd_workspace(int dtype, int64_t n, int64_t V, int64_t D) {
    const int es = bg_elem_size(dtype);
    if (!es || n <= 0 || V <= 0 || D <= 0 || !bwd_sizes_ok(n, V, D)) return 0;
    return bwd_plan(n, V, D, es).bytes;
}

extern "C" int bg_embedding_bwd(int dtype, const void* g, int64_t ldg, const void* ids, int ids_is_64, int64_t n, int64_t D, int64_t V,
                                float scale, void* dw, void* ws, int64_t ws_bytes, bgStream stream) {
    const int es = bg_elem_size(dtype);
    if (!es || n < 0 || D < 0 || V < 0 || ldg < D) return BG_ERR_ARG;
    if (V == 0 || D == 0) return BG_OK;
    if (!dw || (n > 0 && (!g || !ids || !ws))) return BG_ERR_ARG;
    if (!bwd_sizes_ok(n, V, D)) return BG_ERR_SHAPE;
    if (!bg_aligned16(dw) || (n > 0 && !bg_aligned16(ws))) return BG_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    const int64_t bytes = V * D * es, n16 = bytes / 16;
    const BwdPlan p = n > 0 ? bwd_plan(n, V, D, es) : BwdPlan{};
    if (ws_bytes < p.bytes) return BG_ERR_SCRATCH;
    char* base = static_cast<char*>(ws);
    float* part = reinterpret_cast<float*>(base + p.part);
    if (p.few)
        return bg_dispatch_dtype(dtype, [&](auto z) -> int {
            typedef decltype(z) T;
            const T* gg = static_cast<const T*>(g);
            T* d = static_cast<T*>(dw);
            return ids_is_64 ? launch_few<T, true>(p, ids, n, V, gg, ldg, D, scale, d, part, s)
                             : launch_few<T, false>(p, ids, n, V, gg, ldg, D, scale, d, part, s);
        });
    if (bytes % 16) {
        k_fill_tail<<<1, 16, 0, s>>>(static_cast<uint8_t*>(dw) + n16 * 16, (int)(bytes % 16));
        BG_LAUNCH_CHECK();
    }
    if (n == 0) return bg_zero_bytes(dw, n16 * 16, stream);
    int32_t* key[2] = {reinterpret_cast<int32_t*>(base + p.key_a), reinterpret_cast<int32_t*>(base + p.key_b)};
    int32_t* pos[2] = {reinterpret_cast<int32_t*>(base + p.pos_a), reinterpret_cast<int32_t*>(base + p.pos_b)};
    const int32_t *k = key[0], *ps = pos[0];
    if (n <= kSmall) {
        const Fill all{static_cast<uint4*>(dw), n16};
        const int rc = ids_is_64 ? launch_sort_small<0>(p, ids, n, V, key[0], pos[0], all, s)
                                 : launch_sort_small<1>(p, ids, n, V, key[0], pos[0], all, s);
        if (rc != BG_OK) return rc;
    } else {
        int32_t* hist = reinterpret_cast<int32_t*>(base + p.hist);
        int32_t* total = reinterpret_cast<int32_t*>(base + p.total);
        const int64_t share = (n16 + 2 * p.passes - 1) / (2 * p.passes);
        auto fill = [&](int i) {
            const int64_t a = share * i < n16 ? share * i : n16, b = share * (i + 1) < n16 ? share * (i + 1) : n16;
            return Fill{static_cast<uint4*>(dw) + a, b - a};
        };
        for (int q = 0; q < p.passes; ++q) {
            const int o = q & 1, shift = q * p.bits;
            if (q == 0 && ids_is_64) launch_sort_pass<0>(p, ids, nullptr, n, V, shift, hist, total, key[o], pos[o], fill(0), fill(1), s);
            else if (q == 0) launch_sort_pass<1>(p, ids, nullptr, n, V, shift, hist, total, key[o], pos[o], fill(0), fill(1), s);
            else launch_sort_pass<2>(p, key[1 - o], pos[1 - o], n, V, shift, hist, total, key[o], pos[o], fill(2 * q), fill(2 * q + 1), s);
            BG_LAUNCH_CHECK();
        }
        k = key[(p.passes - 1) & 1];
        ps = pos[(p.passes - 1) & 1];
    }
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T* gg = static_cast<const T*>(g);
        T* d = static_cast<T*>(dw);
        const int64_t pieces = (D + Piece<T>::W - 1) / Piece<T>::W;
        const dim3 grid((unsigned)((p.run_tiles + 256 / p.LG - 1) / (256 / p.LG)), (unsigned)((pieces + p.LG - 1) / p.LG));
        const auto kernel = D < Piece<T>::W ? k_embedding_runs<T, true, 0> : p.LG == 64 ? k_embedding_runs<T, false, 64> : k_embedding_runs<T, false, 0>;
        kernel<<<grid, 256, 0, s>>>(k, ps, n, (int32_t)V, gg, ldg, (int)D, scale, d, part, p.C, p.LG);
        BG_LAUNCH_CHECK();
        if (p.run_tiles > 1) {
            k_embedding_join<T><<<dim3((unsigned)p.run_tiles, (unsigned)((D + 255) / 256)), kJoin * kJoinCols, 0, s>>>(k, n, (int32_t)V, part,
                                                                                                                     p.C, D, scale, d);
            BG_LAUNCH_CHECK();
        }
        return BG_OK;
    });
}
