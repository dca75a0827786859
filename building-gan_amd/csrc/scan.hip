// Gated linear recurrence along the rows of each segment, a scan over long sequences, and its backward pass.
//
//   a = sigmoid(gate), c = 1 - a = sigmoid(-gate)          (both from one exponential, each with a relative error of a few units)
//   forward :  h_t = a_t h_{t-1} + c_t x_t                 h before a segment's first row = h0 (or 0)
//   backward:  mu_t = a_t (dh_t + mu_{t+1})                mu after a segment's last row = dlast (or 0)
//              dx_t = c_t (dh_t + mu_{t+1}),  dgate_t = (dh_t + mu_{t+1}) (h_{t-1} - x_t) a_t c_t,  dh0 = mu_first
// Both are chains of maps  s -> A s + B, which compose:  (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2).  A segment's first row
// (its last, for mu) is a CUT: the map that forgets what comes in.  It is marked by A = -1 (a true A is never negative) and
// taken by selection: a product with 0 would let an inf or NaN of another segment through.
//
// Rows are cut into tiles whatever the segments are.  A workgroup reads its tile ONCE, keeps it in registers, composes its
// rows' maps, publishes the tile's map, finds the state that enters the tile from what the tiles before it published, and
// walks its rows from there.  h is never read back: the backward pass rebuilds it from the fp32 state kept at the head of
// every row group, an eighth of the rows.
#include "common.h"

namespace {

// A tile: kThreads / CG row groups of kRows rows times CG column groups of 4 columns; a lane moves 16 bytes (8 bytes) of a
// row of fp32 (16-bit) elements.  CG = 16 (64 columns: one wave can look after a tile's columns), fewer for narrow matrices.
constexpr int kRows = 8;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxCols = 64;
constexpr int kGroup = 8;                        // tiles of a group, groups of a block (see Chain)
constexpr uint32_t kEmpty = 0xFFFFFFFFu;         // what unpublished words hold
constexpr int kSpinLimit = 1 << 22;              // a wait of several seconds: only a workspace in use by another call gets
                                                 // there, and what an empty word gives is a NaN

struct Segs { const int32_t* ptr; int64_t S, N, T; };      // ptr NULL: S segments of T rows

// REV walks the rows upwards: LOGICAL row r is row N - 1 - r, logical segment j is segment S - 1 - j
template <bool REV, bool UNIFORM = false>
__device__ __forceinline__ int64_t seg_lo(const Segs& g, int64_t j) {                // logical first row of logical segment j
    typedef const int32_t __attribute__((address_space(4))) * Scalar;                // (j the same in every lane: a scalar load)
    const int64_t k = REV ? g.S - j : j;
    int64_t p = !g.ptr ? k * g.T : UNIFORM ? (int64_t)((Scalar)(uintptr_t)g.ptr)[k] : (int64_t)g.ptr[k];
    p = p < 0 ? 0 : p > g.N ? g.N : p;
    return REV ? g.N - p : p;
}

// mask[group]: bit i = row i of the group is a segment's first row, bit 8 + i = its last, bit 16 + i = in no segment;
// first[row] / last[row] = that segment where the bit is set; border: any bit at all.  One wave does it.
template <bool REV>
__device__ __forceinline__ void mark_tile(const Segs& g, int64_t row0, int groups, uint32_t* mask, int32_t* first, int32_t* last,
                                          int32_t& border) {
    const int t = threadIdx.x, rows = groups * kRows;
    const int64_t lo_all = seg_lo<REV, true>(g, 0), hi_all = seg_lo<REV, true>(g, g.S), end = row0 + rows;
    const bool inside = lo_all <= row0 && (hi_all >= end || hi_all == g.N);
    for (int k = t; k < groups; k += 64) {
        uint32_t m = 0;
        if (!inside)
            for (int i = 0; i < kRows; ++i) {
                const int64_t r = row0 + k * kRows + i;
                if (r < g.N && (r < lo_all || r >= hi_all)) m |= 0x10000u << i;
            }
        mask[k] = m;
    }
    // how many segments begin at or before row0: scalar loads (the same in every lane), so the search neither waits for the
    // rows of the tile nor makes them wait
    int64_t lo = 0, hi = g.S;
    if (!g.ptr) lo = hi = g.T > 0 ? row0 / g.T + 1 : 0;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (seg_lo<REV, true>(g, mid) <= row0) lo = mid + 1; else hi = mid;
    }
    __builtin_amdgcn_wave_barrier();
    bool found = !inside;
    // nothing to mark where the segment that holds row0 began before it and goes on behind the tile
    const bool plain = lo > 0 && seg_lo<REV, true>(g, lo - 1) < row0 && seg_lo<REV, true>(g, lo) > end;
    for (int64_t j = plain ? g.S : (lo > 0 ? lo - 1 : 0) + t; j < g.S; j += 64) {
        const int64_t a = seg_lo<REV>(g, j), b = seg_lo<REV>(g, j + 1);
        if (a >= end) break;
        if (a >= b) continue;
        const int32_t s = (int32_t)(REV ? g.S - 1 - j : j);
        if (a >= row0) {
            first[a - row0] = s;
            atomicOr(&mask[(a - row0) / kRows], 1u << ((a - row0) % kRows));
            found = true;
        }
        if (b - 1 >= row0 && b - 1 < end) {
            last[b - 1 - row0] = s;
            atomicOr(&mask[(b - 1 - row0) / kRows], 0x100u << ((b - 1 - row0) % kRows));
            found = true;
        }
    }
    found = __any(found);
    if (t == 0) border = found;
}

// The value is computed here and what follows is computed from it: left to itself, the compiler moves the last steps of a
// sigmoid to where its result is used, or keeps products of one walk over the rows for a later one, and either way holds a
// row's worth of registers more than the values it has.
__device__ __forceinline__ void settle(float& v) { asm volatile("" : "+v"(v)); }

// a = sigmoid(g), c = sigmoid(-g) without cancellation: with e = exp(-|g|) <= 1 the smaller one is e / (1 + e), at most 1/2, and
// the larger one is 1 minus it, which is exact to its own rounding: a memory that is long because its a's are near 1 adds up no
// one-sided errors of the reciprocal.  What the rounding of |g| log2(e) leaves out is put back (e * (1 + rest)).  The hardware's
// exponential makes no subnormal numbers: from |g| = 87.4 on the smaller one is 0 (it would be 1.1e-38) and the larger one 1.
// Packed, both are one register: the smaller one with the sign of the gate.
__device__ __forceinline__ float pack_gate(float g) {
    const float m = __builtin_elementwise_minimum(fabsf(g), 110.f);      // (an inf gives no NaN below; a NaN stays one)
    const float p = m * -1.4426950408889634f;
    float e = __builtin_amdgcn_exp2f(p);
    e = fmaf(e, fmaf(p, -0.6931471805599453f, -m), e);
    return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}
__device__ __forceinline__ void gate_pair(float p, float& a, float& c) {
    const float small = fabsf(p), large = 1.f - small;
    const bool low = __float_as_int(p) < 0;
    a = low ? small : large;
    c = low ? large : small;
}
__device__ __forceinline__ void unpack_gate(float& p, float& a, float& c) {
    settle(p);                                       // (or what is taken apart here is kept for the next walk)
    gate_pair(p, a, c);
}

// Four columns of a row as one access at whatever alignment the row has (the hardware takes any; the alignment promised to
// the compiler is the element's)
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[4]; };

// What a thread touches of its tile: a base that is the same in every lane, the byte offset of its first row's piece, and a
// step from row to row (32 bits: the address of an access is one addition).
struct Lane {
    int nv, nrows;                               // columns (0 .. 4) and rows (0 .. kRows) that exist
    __device__ __forceinline__ bool whole() const { return nv == 4 && nrows == kRows; }
};
template <class T>
__device__ __forceinline__ void load_rows(const T* __restrict__ base, uint32_t off, uint32_t step, Lane l, float fill, float (&v)[kRows][4]) {
    const char* p = reinterpret_cast<const char*>(base);
    if (__builtin_expect(l.whole(), 1)) {
        Piece<T> x[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) x[i] = *reinterpret_cast<const Piece<T>*>(p + (uint32_t)(off + i * step));
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = (float)x[i].v[e];
    } else {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[i][e] = i < l.nrows && e < l.nv ? (float)reinterpret_cast<const T*>(p + (uint32_t)(off + i * step))[e] : fill;
    }
}
// Rows as they came from memory: 16-bit elements stay two to a register until they are used
template <class T>
struct Raw {
    Piece<T> v[kRows];
    __device__ __forceinline__ float get(int i, int e) const { return (float)v[i].v[e]; }
};
template <class T>
__device__ __forceinline__ void load_raw(const T* __restrict__ base, uint32_t off, uint32_t step, Lane l, Raw<T>& r) {
    const char* p = reinterpret_cast<const char*>(base);
    if (__builtin_expect(l.whole(), 1)) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) r.v[i] = *reinterpret_cast<const Piece<T>*>(p + (uint32_t)(off + i * step));
    } else {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                r.v[i].v[e] = i < l.nrows && e < l.nv ? reinterpret_cast<const T*>(p + (uint32_t)(off + i * step))[e] : (T)0.f;
    }
}
template <class T>
__device__ __forceinline__ void store_rows(T* __restrict__ base, uint32_t off, uint32_t step, Lane l, const float (&v)[kRows][4]) {
    char* p = reinterpret_cast<char*>(base);
    if (__builtin_expect(l.whole(), 1)) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            Piece<T> x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[e] = bg_round<T>(v[i][e]);
            *reinterpret_cast<Piece<T>*>(p + (uint32_t)(off + i * step)) = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i < l.nrows && e < l.nv) reinterpret_cast<T*>(p + (uint32_t)(off + i * step))[e] = bg_round<T>(v[i][e]);
    }
}
// four columns of fp32 rows of [n, D] (states)
__device__ __forceinline__ void ld_state(const float* __restrict__ p, int64_t row, int64_t D, int64_t c, int nv, float (&v)[4]) {
    if (p && nv == 4) {
        const Piece<float> x = *reinterpret_cast<const Piece<float>*>(p + row * D + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x.v[e];
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = p && e < nv ? p[row * D + c + e] : 0.f;
}
__device__ __forceinline__ void st_state(float* __restrict__ p, int64_t row, int64_t D, int64_t c, int nv, const float (&v)[4]) {
    if (nv == 4) *reinterpret_cast<Piece<float>*>(p + row * D + c) = Piece<float>{{v[0], v[1], v[2], v[3]}};
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < nv) p[row * D + c + e] = v[e];
}

// ------------------------------------------------------------------------------------------------ maps
// The union of the wave's row groups' masks, the same in every lane: loops and branches over borders are the wave's, what a
// lane does there is selection (a divergent branch would keep two copies of the rows).
__device__ __forceinline__ uint32_t wave_mask(uint32_t m, int CG) {
    uint32_t w = 0;
    for (int l = 0; l < 64; l += CG) w |= (uint32_t)__builtin_amdgcn_readlane((int)m, l);
    return w;
}
__device__ __forceinline__ bool bit(uint32_t m, int i) { return (m >> i) & 1; }

struct Map { float A[4], B[4]; };
template <class T>
__device__ __forceinline__ void settle(Piece<T>& x) {
    uint32_t w[sizeof(T)];
    __builtin_memcpy(w, &x, sizeof(w));
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) asm volatile("" : "+v"(w[i]));
    __builtin_memcpy(&x, w, sizeof(w));
}
template <class T>
__device__ __forceinline__ void settle(Raw<T>& r) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) settle(r.v[i]);
}
template <bool CUTS>
__device__ __forceinline__ void after(Map& m, const float (&A1)[4], const float (&B1)[4]) {          // m <- m o (A1, B1)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m.B[e] = CUTS && m.A[e] < 0.f ? m.B[e] : fmaf(m.A[e], B1[e], m.B[e]);
        m.A[e] = CUTS && (m.A[e] < 0.f || A1[e] < 0.f) ? -1.f : m.A[e] * A1[e];
    }
}
__device__ __forceinline__ float apply(float A, float B, float s) { return A < 0.f ? B : fmaf(A, s, B); }

// Maps of the workgroup's row groups: `m` becomes the map of everything before this thread's group (UP: the rows are walked
// from the last group to the first).  In a wave by shuffles (64 / CG groups), then over the waves through LDS.  Returns the
// map of the whole tile in the threads of the LAST group of the walk.  CUTS: the tile has a border (a composition is then
// seven instructions a column instead of two).
struct WaveMaps { float4 A[kWaves][kMaxCols / 4], B[kWaves][kMaxCols / 4]; };
template <bool UP, bool CUTS>
__device__ __forceinline__ Map before_group(Map& m, int CG, int cg, WaveMaps& w) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = UP ? 63 - lane : lane, edge = at / CG;                // this group's place in the wave's walk
    for (int o = 1; o * CG < 64; o <<= 1) {
        float A1[4], B1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            A1[e] = UP ? __shfl_down(m.A[e], o * CG, 64) : __shfl_up(m.A[e], o * CG, 64);
            B1[e] = UP ? __shfl_down(m.B[e], o * CG, 64) : __shfl_up(m.B[e], o * CG, 64);
            if (edge < o) { A1[e] = 1.f; B1[e] = 0.f; }
        }
        after<CUTS>(m, A1, B1);
    }
    if (at >= 64 - CG) {
        w.A[wave][cg] = make_float4(m.A[0], m.A[1], m.A[2], m.A[3]);
        w.B[wave][cg] = make_float4(m.B[0], m.B[1], m.B[2], m.B[3]);
    }
    Map all = m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m.A[e] = UP ? __shfl_down(all.A[e], CG, 64) : __shfl_up(all.A[e], CG, 64);
        m.B[e] = UP ? __shfl_down(all.B[e], CG, 64) : __shfl_up(all.B[e], CG, 64);
        if (edge == 0) { m.A[e] = 1.f; m.B[e] = 0.f; }
    }
    __syncthreads();
    Map pre{{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < kWaves - 1; ++k) {
        const int x = UP ? kWaves - 1 - k : k;
        if (UP ? x > wave : x < wave) {
            const float4 A = w.A[x][cg], B = w.B[x][cg];
            Map y{{A.x, A.y, A.z, A.w}, {B.x, B.y, B.z, B.w}};
            after<CUTS>(y, pre.A, pre.B);
            pre = y;
        }
    }
    after<CUTS>(m, pre.A, pre.B);
    if (UP ? wave == 0 : wave == kWaves - 1) after<CUTS>(all, pre.A, pre.B);
    return all;
}

// ------------------------------------------------------------------------------------------------ from tile to tile
// The tiles of a column block are taken in the order of the walk by a ticket, so whatever a tile waits for belongs to a
// workgroup that already runs (column blocks have nothing to do with each other).  Every tile publishes its map, the last of
// 8 tiles their group's map, the last of 8 groups the STATE behind its 64 tiles: a tile reads at most 7 maps of tiles, 7 of
// groups and one state, and the only chain along the sequence has a link per 64 tiles.  The products are always formed in
// this order, so the bits do not depend on who was first (a look-back that takes the nearest state it finds would).  A word
// is its own flag: (A, B) travel as one 64-bit relaxed atomic, B's bits never being kEmpty; no fences, no other memory is
// ordered by them.
struct Chain {                       // for every column block: tile[group][8][64], group[block][8][64], state[block][64]
    uint64_t *tile, *group;
    uint32_t *state, *ticket, ncb;
};
__device__ __forceinline__ void publish(uint64_t* p, float A, float B) {
    uint32_t b = __float_as_uint(B);
    if (b == kEmpty) b = 0x7FC00000u;                                    // a NaN stays a NaN
    __hip_atomic_store(p, ((uint64_t)b << 32) | __float_as_uint(A), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ bool is_empty(uint64_t v) { return (uint32_t)(v >> 32) == kEmpty; }
// (A, B) <- (A2, B2) o (A, B) for the n words v[0], v[1], ..
__device__ __forceinline__ void then_words(float& A, float& B, const uint64_t (&v)[kGroup - 1], int n) {
#pragma unroll
    for (int i = 0; i < kGroup - 1; ++i)
        if (i < n) {
            const float A2 = __uint_as_float((uint32_t)v[i]), B2 = __uint_as_float((uint32_t)(v[i] >> 32));
            B = apply(A2, B2, B);
            A = A2 < 0.f || A < 0.f ? -1.f : A2 * A;
        }
}
// The first n words of a group, side by side, each asked for until it is there and with a pause between: asking for all
// seven again and again takes from the rows' share of the memory (1,048,576 x 128 fp32 forward 350 us, with this 333 us).
__device__ __forceinline__ void await_words(const uint64_t* p, int n, uint64_t (&v)[kGroup - 1]) {
#pragma unroll
    for (int i = 0; i < kGroup - 1; ++i) v[i] = (uint64_t)kEmpty << 32;
#pragma unroll 1
    for (int k = 0; k < kSpinLimit; ++k) {
        bool wait = false;
#pragma unroll
        for (int i = 0; i < kGroup - 1; ++i)
            if (i < n && __any(is_empty(v[i]))) v[i] = peek(p + i * kMaxCols);
#pragma unroll
        for (int i = 0; i < kGroup - 1; ++i) wait |= i < n && is_empty(v[i]);
        if (!__any(wait)) break;
        __builtin_amdgcn_s_sleep(4);
    }
}

// What enters tile number `k` of the walk, by two waves at once, a lane for each column (a look at another workgroup's word
// takes about a microsecond, and the two levels would be two looks after one another: worth 5 us of 120 at 16,384 x 2,048 bf16
// backward, when that pass had two waves a SIMD).  The first wave publishes the tile's map (ownA, ownB) and composes the maps of its group's tiles before it ..
__device__ __forceinline__ void enter_group(const Chain& ch, uint32_t k, uint32_t cb, uint32_t col, float oA, float oB, float& A, float& B) {
    const int p = (int)(k % kGroup), gp = (int)(k / kGroup % kGroup);
    uint64_t *tiles = ch.tile + ((int64_t)(k / kGroup) * ch.ncb + cb) * (kGroup * kMaxCols) + col;
    A = 1.f;
    B = 0.f;
    if (p < kGroup - 1) publish(tiles + p * kMaxCols, oA, oB);
    if (p > 0) {
        uint64_t v[kGroup - 1];
        await_words(tiles, p, v);
        then_words(A, B, v, p);
    }
    if (p == kGroup - 1 && gp < kGroup - 1)
        publish(ch.group + ((int64_t)(k / (kGroup * kGroup)) * ch.ncb + cb) * (kGroup * kMaxCols) + gp * kMaxCols + col,
                A < 0.f || oA < 0.f ? -1.f : oA * A, apply(oA, oB, B));
}
// .. and the second one finds the state behind the block's groups before that.
__device__ __forceinline__ float enter_block(const Chain& ch, uint32_t k, uint32_t cb, uint32_t col) {
    const int gp = (int)(k / kGroup % kGroup);
    const uint32_t block = k / (kGroup * kGroup);
    const uint64_t *groups = ch.group + ((int64_t)block * ch.ncb + cb) * (kGroup * kMaxCols) + col;
    const uint32_t* before = ch.state + ((int64_t)(block - (block > 0)) * ch.ncb + cb) * kMaxCols + col;
    uint32_t w = block > 0 ? __hip_atomic_load(before, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u;
    float A = 1.f, B = 0.f;
    if (gp > 0) {
        uint64_t v[kGroup - 1];
        await_words(groups, gp, v);
        then_words(A, B, v, gp);
    }
    if (!__all(A < 0.f))                                                 // behind a cut the state from further back is not needed
#pragma unroll 1
        for (int i = 0; i < kSpinLimit && __any(w == kEmpty); ++i) w = __hip_atomic_load(before, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return apply(A, B, __uint_as_float(w));
}

// The next (tile, column block) in the order of the walk; with a single tile there is nothing to order.  false: none left
// (a ticket that another call's workgroups also draw from).  A counter answers about once in 17 ns, so workgroups that start
// together wait for it: 1,024 of the forward pass for 17 us, 768 of the backward pass for 13 us.  So the column blocks are
// dealt out to up to 8 counters, each on a cache line of its own (16,384 x 2,048 bf16 forward 58 us, 73 us with one counter,
// backward 93 and 96 us; 262,144 x 512 bf16 forward 235 and 245 us, backward 336 and 335 us; 100,003 x 333 forward 86 and 94 us).
constexpr uint32_t kTickets = 8, kTicketStep = 32, kXcds = 8;
__device__ __forceinline__ bool take_tile(const Chain& ch, int64_t n_tiles, int64_t& tile, int& cb) {
    __shared__ uint32_t ticket;
    const uint32_t even = (uint32_t)n_tiles / kXcds * kXcds * ch.ncb;    // eight workgroups, one on every XCD, draw from a counter,
    const uint32_t at = (blockIdx.x < even ? blockIdx.x / kXcds : blockIdx.x) % ch.ncb;   // so the counters stay in step
    uint32_t k = blockIdx.x, set = 0, sets = 1;
    if (n_tiles > 1) {
        sets = ch.ncb < kTickets ? ch.ncb : kTickets;
        set = at % sets;
        if (threadIdx.x == 0) ticket = atomicAdd(ch.ticket + set * kTicketStep, 1u);
        __syncthreads();
        k = __builtin_amdgcn_readfirstlane(ticket);                      // addresses of a tile are scalar arithmetic
    }
    const uint32_t size = (ch.ncb - set + sets - 1) / sets;              // column blocks set, set + sets, ..
    tile = k / size;
    cb = (int)(set + k % size * sets);
    return k / size < (uint32_t)n_tiles;
}

__global__ __launch_bounds__(256) void k_scan_clear(uint4* p, int64_t n16, uint4* tickets, int64_t t16) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < t16; i += (int64_t)gridDim.x * 256) tickets[i] = make_uint4(0, 0, 0, 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256)
        p[i] = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
}

// Offset and step of a thread's rows in a matrix of pitch ld, from the tile's lowest row in memory
template <class T, bool REV>
__device__ __forceinline__ uint32_t row_off(int r, int rows, int64_t ld, int c) {
    return ((uint32_t)(REV ? rows - 1 - r : r) * (uint32_t)ld + (uint32_t)c) * (uint32_t)sizeof(T);
}
template <class T, bool REV>
__device__ __forceinline__ uint32_t row_step(int64_t ld) { return (REV ? 0u - (uint32_t)ld : (uint32_t)ld) * (uint32_t)sizeof(T); }

// What the threads of a tile share
struct TileShared {
    int32_t first[2 * kThreads], last[2 * kThreads];                     // kThreads / CG * kRows rows, CG >= 4
    uint32_t mask[kThreads / 4];
    int32_t border;
    WaveMaps wm;
    float4 own[2][kMaxCols / 4], near[2][kMaxCols / 4], far[kMaxCols / 4];
};

// Where a thread stands: rows r0 .. of tile `tile`, four columns from c on
struct Place {
    int RG, cg, rg, r0, rows, cb;
    int64_t row0, c0, c, low;
    Lane l;
};
template <bool REV>
__device__ __forceinline__ Place place(const Segs& g, int64_t D, int CG, int64_t tile, int cb) {
    Place p;
    p.RG = kThreads / CG; p.cg = threadIdx.x & (CG - 1); p.rg = threadIdx.x / CG; p.rows = p.RG * kRows; p.r0 = p.rg * kRows; p.cb = cb;
    p.row0 = tile * p.rows; p.c0 = (int64_t)cb * (CG * 4); p.c = p.c0 + p.cg * 4; p.low = REV ? g.N - p.row0 - p.rows : p.row0;
    const int64_t left = g.N - p.row0 - p.r0;
    p.l.nv = p.c + 4 <= D ? 4 : p.c < D ? (int)(D - p.c) : 0;
    p.l.nrows = left >= kRows ? kRows : left > 0 ? (int)left : 0;
    return p;
}
template <class T, bool REV>
__device__ __forceinline__ void load_tile(const T* __restrict__ m, int64_t ld, const Place& p, float fill, float (&v)[kRows][4]) {
    load_rows(m + p.low * ld + p.c0, row_off<T, REV>(p.r0, p.rows, ld, p.cg * 4), row_step<T, REV>(ld), p.l, fill, v);
}
template <class T, bool REV>
__device__ __forceinline__ void load_tile(const T* __restrict__ m, int64_t ld, const Place& p, Raw<T>& r) {
    load_raw(m + p.low * ld + p.c0, row_off<T, REV>(p.r0, p.rows, ld, p.cg * 4), row_step<T, REV>(ld), p.l, r);
}
template <class T, bool REV>
__device__ __forceinline__ void store_tile(T* __restrict__ m, int64_t ld, const Place& p, const float (&v)[kRows][4]) {
    store_rows(m + p.low * ld + p.c0, row_off<T, REV>(p.r0, p.rows, ld, p.cg * 4), row_step<T, REV>(ld), p.l, v);
}

// The state before this thread's row group, `pre` being the map of the tile's groups before it: through the chain, unless the
// walk is a single tile.  What stands between `ask` and `answer` is done by the other waves while the first two wait.
__device__ __forceinline__ void ask(const Chain& ch, int64_t k, int64_t n_tiles, int64_t D, int CG, const Place& p, bool last_group,
                                    const Map& all, TileShared& sh) {
    if (n_tiles == 1) return;
    if (last_group) {
        sh.own[0][p.cg] = make_float4(all.A[0], all.A[1], all.A[2], all.A[3]);
        sh.own[1][p.cg] = make_float4(all.B[0], all.B[1], all.B[2], all.B[3]);
    }
    __syncthreads();
    const uint32_t col = threadIdx.x & 63;
    if (threadIdx.x < 128 && (int)col < CG * 4 && p.c0 + col < D) {
        if (threadIdx.x < 64) {
            float A, B;
            enter_group(ch, (uint32_t)k, (uint32_t)p.cb, col, (&sh.own[0][0].x)[col], (&sh.own[1][0].x)[col], A, B);
            (&sh.near[0][0].x)[col] = A;
            (&sh.near[1][0].x)[col] = B;
        } else
            (&sh.far[0].x)[col] = enter_block(ch, (uint32_t)k, (uint32_t)p.cb, col);
    }
}
__device__ __forceinline__ void answer(const Chain& ch, int64_t k, int64_t n_tiles, int64_t D, int CG, const Place& p, const Map& pre,
                                       const TileShared& sh, float (&s)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = 0.f;
    if (n_tiles > 1) {
        __syncthreads();
        const uint32_t col = threadIdx.x;
        if (k % (kGroup * kGroup) == kGroup * kGroup - 1 && (int)col < CG * 4 && p.c0 + col < D) {   // the state behind the block
            uint32_t b = __float_as_uint(apply((&sh.own[0][0].x)[col], (&sh.own[1][0].x)[col],
                                               apply((&sh.near[0][0].x)[col], (&sh.near[1][0].x)[col], (&sh.far[0].x)[col])));
            if (b == kEmpty) b = 0x7FC00000u;
            __hip_atomic_store(ch.state + ((int64_t)(k / (kGroup * kGroup)) * ch.ncb + p.cb) * kMaxCols + col, b, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        }
        const float4 A = sh.near[0][p.cg], B = sh.near[1][p.cg], v = sh.far[p.cg];
        s[0] = apply(A.x, B.x, v.x); s[1] = apply(A.y, B.y, v.y); s[2] = apply(A.z, B.z, v.z); s[3] = apply(A.w, B.w, v.w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = apply(pre.A[e], pre.B[e], s[e]);
}

// to[s] = from[s] (or 0) for the segments without rows, dealt out to the tiles' row groups
template <bool REV>
__device__ __forceinline__ void pass_through(const Segs& g, int64_t D, int64_t tile, int64_t n_tiles, const Place& p,
                                             const float* __restrict__ from, float* __restrict__ to) {
    if (!to) return;
    for (int64_t j = tile * p.RG + p.rg; j < g.S; j += n_tiles * p.RG)
        if (seg_lo<REV>(g, j) >= seg_lo<REV>(g, j + 1)) {
            const int64_t s = REV ? g.S - 1 - j : j;
            float v[4];
            ld_state(from, s, D, p.c, p.l.nv, v);
            st_state(to, s, D, p.c, p.l.nv, v);
        }
}

// Borders as a thread sees them: its own row group's first / last rows of segments and rows in no segment, and which rows
// have one in any of the wave's groups (branches are the wave's, what a lane does there is selection).
struct Borders {
    uint32_t m, none, enter, leave, wave_enter, wave_leave;
    __device__ __forceinline__ Borders(const TileShared& sh, const Place& p, int CG, bool border)
        : m(0), none(0), enter(0), leave(0), wave_enter(0), wave_leave(0) {
        if (__builtin_expect(border, 0)) {
            m = sh.mask[p.rg];
            none = m >> 16;
            enter = (m | none) & 0xFF;
            leave = (m >> 8 | none) & 0xFF;
            wave_enter = wave_mask(enter, CG);
            wave_leave = wave_mask(leave, CG);
        }
    }
    // before the next walk over the rows: or the compiler keeps the tests of 8 rows' bits, a register each
    __device__ __forceinline__ void again() {
        asm volatile("" : "+v"(m), "+v"(none), "+v"(enter), "+v"(leave));
    }
};
// s <- the state before row i of the group where a segment begins there (0 where the row is in none)
__device__ __forceinline__ void enter_row(const Borders& w, int i, const TileShared& sh, const Place& p, const float* __restrict__ h0, int64_t D,
                                          float (&s)[4]) {
    const bool seg = bit(w.m, i);
    float s0[4];
    ld_state(seg ? h0 : nullptr, seg ? sh.first[p.r0 + i] : 0, D, p.c, p.l.nv, s0);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = bit(w.enter, i) ? s0[e] : s[e];
}

// Row i of the group from above: where a segment ends there (or the row is in none) nothing comes in, s <- 0, and the gradient
// d of its h takes that of the segment's last state (or is 0)
__device__ __forceinline__ void leave_row(const Borders& w, int i, const TileShared& sh, const Place& p, const float* __restrict__ dlast,
                                          int64_t D, float (&d)[4], float (&s)[4]) {
    const bool seg = bit(w.m, 8 + i);
    float ds[4];
    ld_state(seg ? dlast : nullptr, seg ? sh.last[p.r0 + i] : 0, D, p.c, p.l.nv, ds);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        d[e] = bit(w.none, i) ? 0.f : d[e] + ds[e];
        s[e] = bit(w.leave, i) ? 0.f : s[e];
    }
}

// ------------------------------------------------------------------------------------------------ forward
// x and gate are read once, h (and an eighth of it in fp32) written once.  fp32 rows are bound by memory: 1,048,576 x 128
// 332 us, 4.85 TB/s, what a copy of 4 GiB reaches (4.81).  16-bit rows carry half the bytes for the same arithmetic, about
// 33 instructions an element: 262,144 x 512 bf16 230 us (3.5 TB/s), of which the SIMDs issue for half; without the look-back
// the same rows took 186 us, what remains of it is a tile's wait of some 3 us that four waves a SIMD do not hide.  Rows that
// begin at any address are read almost twice (100,003 x 333 fp16: 262 MB for 133), but that is not what they cost: at a pitch of
// 384 it is 165 MB and the same 95 us.  The last column block is: 320 columns take 67 us, so its 13 columns cost as much as two
// full blocks.  In narrow rows a load instruction of a wave touches 16 pieces of 32 bytes, 256 bytes apart: 1,048,576 x 16 bf16
// 52 us where its 110 MB would take 23.  The bound of 128 registers (four waves instead of three) was worth 273 -> 247 us at
// 262,144 x 512 bf16; five would take spills.
template <class T, bool REV>
__global__ __launch_bounds__(kThreads, 4) void k_scan_fwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg, Segs g,
                                                       int64_t D, const float* __restrict__ h0, int CG, Chain ch, int64_t n_tiles,
                                                       T* __restrict__ h, int64_t ldh, float* __restrict__ h_last, float* __restrict__ heads) {
    __shared__ TileShared sh;
    int64_t tile;
    int cb;
    if (!take_tile(ch, n_tiles, tile, cb)) return;
    const Place p = place<REV>(g, D, CG, tile, cb);
    if (threadIdx.x < 64) mark_tile<REV>(g, p.row0, p.RG, sh.mask, sh.first, sh.last, sh.border);
    float a[kRows][4], b[kRows][4];                                      // a row's map: s -> a s + b, b = c x
    load_tile<T, REV>(gate, ldg, p, __builtin_inff(), a);                // where there is no row: a = 1, b = 0, the map that
    load_tile<T, REV>(x, ldx, p, 0.f, b);                                // changes nothing
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float ce;
            gate_pair(pack_gate(a[i][e]), a[i][e], ce);
            b[i][e] *= ce;
            settle(a[i][e]);
            settle(b[i][e]);
        }
    __syncthreads();
    const bool border = __builtin_amdgcn_readfirstlane(sh.border) != 0;
    Borders w(sh, p, CG, border);
    Map f{{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (bit(w.wave_enter, i)) {
            enter_row(w, i, sh, p, h0, D, f.B);
#pragma unroll
            for (int e = 0; e < 4; ++e) {                                // a row in no segment: 0, whatever it holds
                a[i][e] = bit(w.none, i) ? 0.f : a[i][e];
                b[i][e] = bit(w.none, i) ? 0.f : b[i][e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.B[e] = fmaf(a[i][e], f.B[e], b[i][e]);
            f.A[e] *= a[i][e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) f.A[e] = w.enter ? -1.f : f.A[e];
    const Map all = border ? before_group<false, true>(f, CG, p.cg, sh.wm) : before_group<false, false>(f, CG, p.cg, sh.wm);
    float s[4];
    ask(ch, tile, n_tiles, D, CG, p, p.rg == p.RG - 1, all, sh);
    w.again();
    answer(ch, tile, n_tiles, D, CG, p, f, sh, s);
    if (heads && p.l.nrows > 0) st_state(heads, tile * p.RG + p.rg, D, p.c, p.l.nv, s);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (bit(w.wave_enter, i)) enter_row(w, i, sh, p, h0, D, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[i][e] = s[e] = fmaf(a[i][e], s[e], b[i][e]);
        if (bit(w.wave_leave, i) && h_last && bit(w.m, 8 + i)) st_state(h_last, sh.last[p.r0 + i], D, p.c, p.l.nv, s);
    }
    store_tile<T, REV>(h, ldh, p, b);
    pass_through<REV>(g, D, tile, n_tiles, p, h0, h_last);
}

// ------------------------------------------------------------------------------------------------ backward
// The walk for mu goes from the last tile to the first.  h before a row group was kept by the forward pass, so
// q = (h_before - x) a c is made while the tile's state is asked for; per element a, c, dh and q stay: dx = c lam,
// dgate = q lam.  Three waves a SIMD hide the loads' and the look-back's latency, so registers are what counts: a and c in one,
// x and dh as they came, nothing kept from one walk over the rows for the next (133 registers for 16-bit rows, 163 for fp32).
// 1,048,576 x 128 fp32 527 us (5.1 TB/s; a and c apart, two waves: 553 us), 262,144 x 512 bf16 342 us (3.9 TB/s; apart, two
// waves: 436 us; four waves by spilling ten registers: 346 us).
template <class T, bool REV>
__global__ __launch_bounds__(kThreads, 3) void k_scan_bwd(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg,
                                                       const T* __restrict__ dh, int64_t lddh, const float* __restrict__ dlast, Segs g,
                                                       int64_t D, const float* __restrict__ h0, int CG, Chain ch, int64_t n_tiles,
                                                       const float* __restrict__ heads, T* __restrict__ dx, int64_t lddx,
                                                       T* __restrict__ dgate, int64_t lddg, float* __restrict__ dh0) {
    __shared__ TileShared sh;
    int64_t k;
    int cb;
    if (!take_tile(ch, n_tiles, k, cb)) return;
    const int64_t tile = n_tiles - 1 - k;
    const Place p = place<REV>(g, D, CG, tile, cb);
    if (threadIdx.x < 64) mark_tile<REV>(g, p.row0, p.RG, sh.mask, sh.first, sh.last, sh.border);
    float ac[kRows][4], q[kRows][4], s[4];                               // ac: the gates as read, then a and c, then dx
    Raw<T> xr, dr;
    load_tile<T, REV>(gate, ldg, p, __builtin_inff(), ac);
    if (dh) load_tile<T, REV>(dh, lddh, p, dr);
    else
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) dr.v[i].v[e] = (T)0.f;
    ld_state(heads, tile * p.RG + p.rg, D, p.c, p.l.nrows > 0 ? p.l.nv : 0, s);
    load_tile<T, REV>(x, ldx, p, xr);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ac[i][e] = pack_gate(ac[i][e]);
            settle(ac[i][e]);
        }
    settle(dr);
    settle(xr);
    __syncthreads();
    const bool border = __builtin_amdgcn_readfirstlane(sh.border) != 0;
    Borders w(sh, p, CG, border);
    Map u{{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i) {
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = dr.get(i, e);
        if (bit(w.wave_leave, i)) leave_row(w, i, sh, p, dlast, D, d, u.B);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, c;
            unpack_gate(ac[i][e], a, c);
            u.B[e] = a * (d[e] + u.B[e]);
            u.A[e] *= a;
        }
    }
    settle(dr);
    settle(xr);
    w.again();
#pragma unroll
    for (int e = 0; e < 4; ++e) u.A[e] = w.leave ? -1.f : u.A[e];
    const Map all = border ? before_group<true, true>(u, CG, p.cg, sh.wm) : before_group<true, false>(u, CG, p.cg, sh.wm);
    ask(ch, k, n_tiles, D, CG, p, p.rg == 0, all, sh);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (bit(w.wave_enter, i)) enter_row(w, i, sh, p, h0, D, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float xi = xr.get(i, e), hb = s[e];
            float a, c;
            unpack_gate(ac[i][e], a, c);
            s[e] = fmaf(a, hb, c * xi);
            q[i][e] = (hb - xi) * (a * c);
            settle(q[i][e]);
        }
    }
    w.again();
    answer(ch, k, n_tiles, D, CG, p, u, sh, s);
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i) {
        float d[4];
        settle(dr.v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = dr.get(i, e);
        if (bit(w.wave_leave, i)) leave_row(w, i, sh, p, dlast, D, d, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lam = d[e] + s[e];
            float a, c;
            unpack_gate(ac[i][e], a, c);
            ac[i][e] = c * lam;
            q[i][e] *= lam;
            s[e] = a * lam;
        }
        if (bit(w.wave_enter, i)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {                                // rows in no segment: 0, whatever they hold
                ac[i][e] = bit(w.none, i) ? 0.f : ac[i][e];
                q[i][e] = bit(w.none, i) ? 0.f : q[i][e];
            }
            if (bit(w.m, i) && dh0) st_state(dh0, sh.first[p.r0 + i], D, p.c, p.l.nv, s);
        }
    }
    store_tile<T, REV>(dx, lddx, p, ac);
    store_tile<T, REV>(dgate, lddg, p, q);
    pass_through<REV>(g, D, tile, n_tiles, p, dlast, dh0);
}

// ------------------------------------------------------------------------------------------------ one row per segment
// A launch's latency: 2.4 us at 50 x 256 fp32.
template <class T, int W>
__global__ __launch_bounds__(256) void k_scan_step(const T* __restrict__ x, int64_t ldx, const T* __restrict__ gate, int64_t ldg,
                                                   const float* state, int64_t lds_, int64_t D, T* __restrict__ h, int64_t ldh,
                                                   float* state_out, int64_t ldso) {
    const int64_t row = blockIdx.x;
    const int64_t c0 = ((int64_t)blockIdx.y * 256 + threadIdx.x) * W;
    if (c0 >= D) return;
    const BgVec<T, W> xv = *reinterpret_cast<const BgVec<T, W>*>(x + row * ldx + c0);
    const BgVec<T, W> gv = *reinterpret_cast<const BgVec<T, W>*>(gate + row * ldg + c0);
    BgVec<float, W> sv = *reinterpret_cast<const BgVec<float, W>*>(state + row * lds_ + c0);
    BgVec<T, W> hv;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        float a, c;
        gate_pair(pack_gate((float)gv.v[e]), a, c);
        sv.v[e] = fmaf(a, sv.v[e], c * (float)xv.v[e]);
        hv.v[e] = bg_round<T>(sv.v[e]);
    }
    *reinterpret_cast<BgVec<T, W>*>(h + row * ldh + c0) = hv;
    *reinterpret_cast<BgVec<float, W>*>(state_out + row * ldso + c0) = sv;
}

// ------------------------------------------------------------------------------------------------ host side
int column_groups(int64_t D) { return D > 32 ? 16 : D > 16 ? 8 : 4; }
int64_t tiles_of(int64_t n, int64_t D) {
    const int64_t rows = kThreads * kRows / column_groups(D);
    return (n + rows - 1) / rows;
}
unsigned column_blocks(int64_t D) { return (unsigned)((D + 4 * column_groups(D) - 1) / (4 * column_groups(D))); }

template <class T>
bool piece_ok(const void* p, int64_t ld, int64_t D) {
    return D % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
}

int check_scan(int dtype, int64_t n, int64_t D, int64_t S, const int32_t* rowptr) {
    if (!bg_elem_size(dtype) || n < 0 || D < 0 || S < 0) return BG_ERR_ARG;
    if (!rowptr && (S == 0 ? n != 0 : n % S != 0)) return BG_ERR_ARG;
    if (n > INT32_MAX || S >= INT32_MAX || D > (1 << 20)) return BG_ERR_SHAPE;
    if (D > 0 && tiles_of(n, D) > (int64_t)(UINT32_MAX / kThreads) / column_blocks(D)) return BG_ERR_SHAPE;   // work-items < 2^32
    return BG_OK;
}
bool pitch_ok(int64_t ld) { return ld <= (1 << 21); }      // a tile's offsets (at most 512 rows) fit 32 bits, in bytes too

struct ScanWs { int64_t tile, group, state, ticket, bytes; };
ScanWs scan_ws(int64_t n, int64_t D) {
    const int64_t t = tiles_of(n, D);
    ScanWs w;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    const int64_t blocks = t / (kGroup * kGroup) + 1, lane = column_blocks(D) * kMaxCols;
    w.tile = take(8 * (t / kGroup + 1) * kGroup * lane);
    w.group = take(8 * blocks * kGroup * lane);
    w.state = take(4 * blocks * lane);
    w.ticket = take(4 * kTicketStep * kTickets);
    w.bytes = at;
    return w;
}
// the words of `tiles` tiles emptied, the tickets at zero
Chain make_chain(void* ws, int64_t n, int64_t D, int64_t tiles, hipStream_t s) {
    const ScanWs w = scan_ws(n, D);
    char* base = static_cast<char*>(ws);
    const Chain ch{reinterpret_cast<uint64_t*>(base + w.tile), reinterpret_cast<uint64_t*>(base + w.group),
                   reinterpret_cast<uint32_t*>(base + w.state), reinterpret_cast<uint32_t*>(base + w.ticket), column_blocks(D)};
    if (tiles > 1) k_scan_clear<<<bg_grid_for(w.ticket / 16, 256 * 4, 2048), 256, 0, s>>>(static_cast<uint4*>(ws), w.ticket / 16,
                                                                                            reinterpret_cast<uint4*>(ch.ticket), (w.bytes - w.ticket) / 16);
    return ch;
}

template <class T, bool REV>
void launch_scan_fwd(const T* x, int64_t ldx, const T* gate, int64_t ldg, Segs g, int64_t D, const float* h0, void* ws, T* h, int64_t ldh,
                     float* h_last, float* heads, hipStream_t s) {
    const int64_t tiles = tiles_of(g.N, D);
    const Chain ch = make_chain(ws, g.N, D, tiles, s);
    k_scan_fwd<T, REV><<<(unsigned)tiles * column_blocks(D), kThreads, 0, s>>>(x, ldx, gate, ldg, g, D, h0, column_groups(D), ch, tiles, h,
                                                                                   ldh, h_last, heads);
}
template <class T, bool REV>
void launch_scan_bwd(const T* x, int64_t ldx, const T* gate, int64_t ldg, const T* dh, int64_t lddh, const float* dlast, Segs g, int64_t D,
                     const float* h0, void* ws, const float* heads, T* dx, int64_t lddx, T* dgate, int64_t lddg, float* dh0, hipStream_t s) {
    const int64_t tiles = tiles_of(g.N, D);
    const Chain ch = make_chain(ws, g.N, D, tiles, s);
    k_scan_bwd<T, REV><<<(unsigned)tiles * column_blocks(D), kThreads, 0, s>>>(x, ldx, gate, ldg, dh, lddh, dlast, g, D, h0,
                                                                                   column_groups(D), ch, tiles, heads, dx, lddx, dgate, lddg, dh0);
}

__global__ __launch_bounds__(256) void k_copy_or_zero(const float* __restrict__ src, float* __restrict__ dst, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = src ? src[i] : 0.f;
}

}  // namespace

extern "C" int64_t bg_gated_scan_heads(int64_t n_rows, int64_t D) { return n_rows > 0 && D > 0 ? tiles_of(n_rows, D) * (kThreads / column_groups(D)) * D : 0; }

extern "C" int64_t bg_gated_scan_workspace(int64_t n_rows, int64_t D) { return n_rows > 0 && D > 0 ? scan_ws(n_rows, D).bytes : 0; }

extern "C" int bg_gated_scan_fwd(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const int32_t* rowptr, int64_t n_seg,
                                 int64_t n_rows, int64_t D, const float* h0, int reverse, void* h, int64_t ldh, float* h_last,
                                 float* heads, void* ws, int64_t ws_bytes, bgStream stream) {
    const int rc = check_scan(dtype, n_rows, D, n_seg, rowptr);
    if (rc != BG_OK) return rc;
    if (ldx < D || ldg < D || ldh < D) return BG_ERR_ARG;
    if (!pitch_ok(ldx) || !pitch_ok(ldg) || !pitch_ok(ldh)) return BG_ERR_SHAPE;
    if (D == 0) return BG_OK;
    hipStream_t s = (hipStream_t)stream;
    if (n_rows == 0) {                                     // no rows: the states pass through
        if (!h_last || n_seg == 0) return BG_OK;
        k_copy_or_zero<<<bg_grid_for(n_seg * D, 256, 4096), 256, 0, s>>>(h0, h_last, n_seg * D);
        BG_LAUNCH_CHECK();
        return BG_OK;
    }
    if (!x || !gate || !h || !ws) return BG_ERR_ARG;
    if (!bg_aligned16(ws)) return BG_ERR_ALIGN;
    if (ws_bytes < scan_ws(n_rows, D).bytes) return BG_ERR_SCRATCH;
    const Segs g{rowptr, n_seg, n_rows, rowptr ? 0 : n_rows / n_seg};
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate);
        T* hh = static_cast<T*>(h);
        if (reverse) launch_scan_fwd<T, true>(xx, ldx, gg, ldg, g, D, h0, ws, hh, ldh, h_last, heads, s);
        else launch_scan_fwd<T, false>(xx, ldx, gg, ldg, g, D, h0, ws, hh, ldh, h_last, heads, s);
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}

extern "C" int bg_gated_scan_bwd(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const void* dh, int64_t lddh,
                                 const float* dlast, const int32_t* rowptr, int64_t n_seg, int64_t n_rows, int64_t D, const float* h0,
                                 int reverse, const float* heads, void* dx, int64_t lddx, void* dgate, int64_t lddg, float* dh0, void* ws,
                                 int64_t ws_bytes, bgStream stream) {
    const int rc = check_scan(dtype, n_rows, D, n_seg, rowptr);
    if (rc != BG_OK) return rc;
    if (ldx < D || ldg < D || (dh && lddh < D) || lddx < D || lddg < D) return BG_ERR_ARG;
    if (!pitch_ok(ldx) || !pitch_ok(ldg) || (dh && !pitch_ok(lddh)) || !pitch_ok(lddx) || !pitch_ok(lddg)) return BG_ERR_SHAPE;
    if (D == 0) return BG_OK;
    hipStream_t s = (hipStream_t)stream;
    if (n_rows == 0) {
        if (!dh0 || n_seg == 0) return BG_OK;
        k_copy_or_zero<<<bg_grid_for(n_seg * D, 256, 4096), 256, 0, s>>>(dlast, dh0, n_seg * D);
        BG_LAUNCH_CHECK();
        return BG_OK;
    }
    if (!x || !gate || !heads || !dx || !dgate || !ws) return BG_ERR_ARG;
    if (!bg_aligned16(ws)) return BG_ERR_ALIGN;
    if (ws_bytes < scan_ws(n_rows, D).bytes) return BG_ERR_SCRATCH;
    const Segs g{rowptr, n_seg, n_rows, rowptr ? 0 : n_rows / n_seg};
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate), *dd = static_cast<const T*>(dh);
        T *ox = static_cast<T*>(dx), *og = static_cast<T*>(dgate);
        if (reverse) launch_scan_bwd<T, true>(xx, ldx, gg, ldg, dd, lddh, dlast, g, D, h0, ws, heads, ox, lddx, og, lddg, dh0, s);
        else launch_scan_bwd<T, false>(xx, ldx, gg, ldg, dd, lddh, dlast, g, D, h0, ws, heads, ox, lddx, og, lddg, dh0, s);
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}

extern "C" int bg_gated_scan_step(int dtype, const void* x, int64_t ldx, const void* gate, int64_t ldg, const float* state, int64_t lds,
                                  int64_t n, int64_t D, void* h, int64_t ldh, float* state_out, int64_t ldso, bgStream stream) {
    if (!bg_elem_size(dtype) || n < 0 || D < 0 || ldx < D || ldg < D || lds < D || ldh < D || ldso < D) return BG_ERR_ARG;
    if (n == 0 || D == 0) return BG_OK;
    if (!x || !gate || !state || !h || !state_out) return BG_ERR_ARG;
    if (n * 256 > UINT32_MAX || D > (1 << 20)) return BG_ERR_SHAPE;
    return bg_dispatch_dtype(dtype, [&](auto z) -> int {
        typedef decltype(z) T;
        const T *xx = static_cast<const T*>(x), *gg = static_cast<const T*>(gate);
        T* hh = static_cast<T*>(h);
        const bool wide = piece_ok<T>(x, ldx, D) && piece_ok<T>(gate, ldg, D) && piece_ok<T>(h, ldh, D) && piece_ok<float>(state, lds, D) &&
                          piece_ok<float>(state_out, ldso, D);
        const dim3 grid((unsigned)n, (unsigned)((D + (wide ? 1023 : 255)) / (wide ? 1024 : 256)));
        if (wide) k_scan_step<T, 4><<<grid, 256, 0, (hipStream_t)stream>>>(xx, ldx, gg, ldg, state, lds, D, hh, ldh, state_out, ldso);
        else k_scan_step<T, 1><<<grid, 256, 0, (hipStream_t)stream>>>(xx, ldx, gg, ldg, state, lds, D, hh, ldh, state_out, ldso);
        BG_LAUNCH_CHECK();
        return BG_OK;
    });
}
