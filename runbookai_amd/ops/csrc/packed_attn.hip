// Causal attention of packed sequences with its gradients, for training
// (gfx950): bf16, grouped heads, head dim 64 or 128.
//
// With s_ij = scale q_i.k_j over the places j <= i of i's own sequence:
//   forward    P_ij = exp(s_ij) / l_i,  l_i = sum_j exp(s_ij),  o_i = sum_j P_ij v_j
//   backward   dP_ij = do_i.v_j,  delta_i = sum_j P_ij dP_ij = do_i.o_i
//              dS_ij = P_ij (dP_ij - delta_i)
//              dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,
//              dv_j = sum_i P_ij do_i          (dk, dv also over the group's heads)
// P is recomputed from q, k and the row's log-sum in the backward pass.
//
// Every product is a v_mfma_f32_32x32x16_bf16.  Its fragments, for lane l with
// c = l & 31, hi = l >> 5:
//   A[32x16]: j=0..7 -> A[c][8 hi + j]      B[16x32]: j -> B[8 hi + j][c]
//   C[32x32]: r=0..15 -> C[(r & 3) + 8 (r >> 2) + 4 hi][c]
// The sum over k may run in any order that A and B share.  Taking
//   k' = 16 s + 4 hi + (j & 3) + 8 (j >> 2)   for slice s, element j,
// the C registers 8s..8s+7 of one product ARE the B fragment of slice s of the
// next, in place: P and dS never leave their lane, neither through LDS nor
// across lanes.  So each chain is laid out with the shared index on C's rows:
//   forward  S^T = K Q^T -> O^T += V^T P^T
//   dq       S^T = K Q^T, dP^T = V dO^T -> dQ^T += K^T dS^T
//   dk, dv   S = Q K^T, dP = dO V^T -> dV^T += dO^T P, dK^T += Q^T dS
// and the other operand (V^T, K^T, dO^T, Q^T) is read from its row-major LDS
// tile by ds_read_b64_tr_b16: of a group of 16 lanes, lane i passes the
// address of 4 elements of row i/4 and receives column i of the 4 rows.  With
// the softmax statistics on the columns, each lane keeps its own row's.
//
// dq and (dk, dv) are two kernels that both recompute P: 7 products where one
// pass would need 5, but no atomics, so the same inputs give the same bits.
//
// Precision: scores, statistics, delta and all sums are fp32; P and dS are
// rounded to bf16 as operands of a product, which bf16 inputs ask for anyway.
// delta_i = do_i.o_i inherits o's errors, and where dP - delta cancels (rows
// that attend to few places) they show in dq and dk.  So the forward pass also
// keeps what o's rounding left over (out_lo, as bf16), which takes the rounding
// out of delta; and the first tile of each sequence, whose rows have few places
// to attend to, takes delta_i = sum_j P_ij dP_ij in fp32, by a sweep of its own
// over its (at most 128) keys.  Of the policy's batch, dq is then 1.46 times as
// far from exact as its own rounding alone; from the rounded o it was 1.50.
#include "common.h"

#include "packed_attn.h"

#include <type_traits>

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int int4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

#define ROWS PACKED_ROWS
#define LOG2E 1.4426950408889634f

namespace {

DEVINL f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

DEVINL f32x16_t zero16() {
    f32x16_t z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// C-fragment row of register r
DEVINL int crow(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }

// Registers 8s..8s+7 of a C fragment, rounded, as the B fragment of slice s.
DEVINL bf16x8_t pack8(const f32x16_t& c, int s) {
    union { bf16x2_t h[4]; bf16x8_t v; } u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        u.h[j] = __builtin_convertvector((float2_t{c[8 * s + 2 * j], c[8 * s + 2 * j + 1]}),
                                         bf16x2_t);
    return u.v;
}

// x, for a branch that few waves take and that begins with it: keeps the
// compiler from making selects of the branch that all waves run.
DEVINL int seldom(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// LDS tile of rows of D bf16, in 16-byte chunks, chunk c of row r at
// c ^ turn(r).  This spreads both kinds of reads over all 64 banks: 16 lanes
// with the same chunk of 16 rows (16 bytes each), and 32 lanes with 64 bytes of
// 4 rows each (8 bytes each).
template <int D>
DEVINL unsigned turn(unsigned row) {
    return D == 128 ? ((row & 3u) << 2) | ((row >> 2) & 3u)
                    : (((row >> 1) & 1u) << 2) | ((row >> 2) & 3u);
}

// Where a lane's parts of a tile begin.  `turn` and the position in a row only
// meet in exclusive-ors, so all fragments are one exclusive-or with a constant
// away from one address for each kind of read: `rows` for a fragment of rows,
// `cols` for one of the transpose.  Where registers allow (KEPT), each of these is
// kept, and which tile is meant goes into the reads' constant offsets; else they
// are made anew from two every step (`fresh`), or the compiler would keep them.
// (8192 rows forward: 539 us kept, 551 made anew; dq of 8192 packed: 309, 313.)
template <int D, bool KEPT>
struct Lane {
    static constexpr int N = KEPT ? D / 16 : 1;
    unsigned rows[N], cols[N];
    DEVINL explicit Lane(int lane) {
        const unsigned r = lane & 31, hi = lane >> 5, i = lane & 15, c = 4 * hi + (i >> 2);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            rows[n] = (r * (D * 2) + ((hi ^ turn<D>(r)) << 4)) ^ (n << 5);
            cols[n] = (c * (D * 2) + 8 * (i & 1) +
                       (((2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ turn<D>(c)) << 4)) ^ (n << 5);
            if (KEPT) asm volatile("" : "+v"(rows[n]), "+v"(cols[n]));
        }
    }
    DEVINL Lane fresh(unsigned tile) const {
        Lane l = *this;
        if (!KEPT) {
            l.rows[0] += tile;
            l.cols[0] += tile;
            asm volatile("" : "+v"(l.rows[0]), "+v"(l.cols[0]));
        }
        return l;
    }
    DEVINL unsigned row(int n) const { return KEPT ? rows[n % N] : rows[0] ^ (n << 5); }
    DEVINL unsigned col(int n) const { return KEPT ? cols[n % N] : cols[0] ^ (n << 5); }
};

// A fragment of 32 rows from `tile`, columns 16 s..16 s+15
template <typename L>
DEVINL bf16x8_t rows_frag(const char* tile, const L& l, int s) {
    return *reinterpret_cast<const bf16x8_t*>(tile + l.row(s));
}

// A fragment of the transpose: columns 32 db..32 db+31 as its rows, and the
// rows k' (as above, slice 0) from `tile` as its columns
template <int D, typename L>
DEVINL bf16x8_t cols_frag(char* tile, const L& l, int db) {
    union { short4_t h[2]; bf16x8_t v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(tile + l.col(2 * db)));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(   // 8 rows on
        (lds_short4_t*)(tile + l.col(2 * db + 1) + 16 * D));
    return u.v;
}

// Keeps what is written before it before what is written behind it.  With D 128
// the kernels read some fragments ahead of the products that take them, and put
// the softmax between products; the compiler alone reads each pair of fragments
// right before its products (dq 322 against 311 us).  With D 64 four waves a SIMD
// cover for each other, and there are no registers to read ahead.
template <int D>
DEVINL void in_order() { if (D == 128) __builtin_amdgcn_sched_barrier(0); }

// The first of a fragment's 16 elements whose exp goes beneath product i of n:
// none beneath the first, while the product that makes them ends.
DEVINL constexpr int beneath(int i, int n) { return i ? (i - 1) * 16 / (n - 1) : 0; }

// Moves N rows from global memory straight into an LDS tile, 16 bytes a lane,
// by a workgroup of THREADS.  A wave's lanes fill consecutive chunks, so the
// order of chunks in a row (`turn`) is made by which chunk a lane reads.  A row
// past `last` is read as row `last` instead: what it holds has P = 0.  Nothing
// lands in a register, so the compiler need not know of the load; arrived()
// waits for it.
template <int D, int N, int THREADS>
struct Mover {
    static constexpr int STEP = THREADS / (D / 8);   // rows that the workgroup moves at a time
    static constexpr int LOADS = N / STEP;           // that each wave issues for a tile
    static_assert(STEP % 16 == 0 && N % STEP == 0, "turn(row + STEP) is turn(row)");
    int row;
    unsigned chunk, off, wave;
    long pitch;   // bytes from row to row
    DEVINL explicit Mover(long stride) {
        row = threadIdx.x / (D / 8);
        chunk = ((threadIdx.x % (D / 8)) ^ turn<D>(row)) * 16;
        pitch = stride * 2;
        off = row * (unsigned)pitch + chunk;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) * (WAVE * 16);
    }
    DEVINL const char* at(const ushort_t* base, int row) const {
        return reinterpret_cast<const char*>(base) + row * pitch;
    }
    DEVINL static void issue(unsigned to, unsigned at, const char* from) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(to), "v"(at), "s"(from)
                     : "memory", "m0");
    }
    // from row 0 of the tile on, which ends with row `last`
    DEVINL void move(const char* from, int last, char* tile) const {
        const unsigned to =
            (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)tile + wave;
        if (N - 1 <= last) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                issue(to + i * STEP * D * 2, off, from + i * STEP * pitch);
        } else {
            const int r = seldom(row);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                issue(to + i * STEP * D * 2,
                      __umul24(min(r + i * STEP, last), (unsigned)pitch) + chunk, from);
        }
    }
};

// 64 floats, one a lane: `from[i]` of each lane's own i
DEVINL void move64(const float* from, int i, const float* to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(
                       (unsigned)(unsigned long)(__attribute__((address_space(3))) const float*)to)),
                   "v"((unsigned)i * 4u), "s"(from)
                 : "memory", "m0");
}

// All of the wave's own moves but its last N are in LDS (loads end in the order
// of their issue); a barrier must follow.
template <int N = 0>
DEVINL void arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// One row's values as a B fragment set: B[k][c] = x[row of lane c][k]
template <int D>
DEVINL void load_row(bf16x8_t (&f)[D / 16], const ushort_t* row, bool real, int hi) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        f[s] = bf16x8_t{};
        if (real) f[s] = *reinterpret_cast<const bf16x8_t*>(row + s * 16 + hi * 8);
    }
}

// Waits for the loads of f here.  Otherwise the compiler waits at f's first use
// in the loop, each time round, and with it for the tiles on their way.
template <int N>
DEVINL void settle(bf16x8_t (&f)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

// x's sum, or maximum, over a lane and its partner in the other half of the wave
DEVINL float both_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                    false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
DEVINL float both_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                    false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Writes a transposed accumulator's column (the lane's row) times `factor`;
// `rest` (may be null) gets what the rounding to bf16 left over.  A lane and its
// partner hold 4 elements each of every 8: they swap halves of two groups, so
// that each writes 16 bytes of one.
template <int D>
DEVINL void store_row(const f32x16_t (&acc)[D / 32], float factor, ushort_t* row, int hi,
                      ushort_t* rest, bool mine) {
    union Pair { bf16x2_t h; unsigned u; };
    typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
    auto join = [](Pair a0, Pair a1, Pair b0, Pair b1) {
        const auto r0 = __builtin_amdgcn_permlane32_swap(a0.u, b0.u, false, false);
        const auto r1 = __builtin_amdgcn_permlane32_swap(a1.u, b1.u, false, false);
        return uint4_t{r0[0], r1[0], r0[1], r1[1]};
    };
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            Pair x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2_t v = {acc[db][4 * g + 2 * i] * factor,
                                    acc[db][4 * g + 2 * i + 1] * factor};
                x[i].h = __builtin_convertvector(v, bf16x2_t);
                const float2_t left = {v[0] - (float)x[i].h[0], v[1] - (float)x[i].h[1]};
                y[i].h = __builtin_convertvector(left, bf16x2_t);
            }
            const int at = db * 32 + 8 * (g + hi);
            const uint4_t a = join(x[0], x[1], x[2], x[3]);
            if (mine) *reinterpret_cast<uint4_t*>(row + at) = a;
            if (rest) {
                const uint4_t b = join(y[0], y[1], y[2], y[3]);
                if (mine) *reinterpret_cast<uint4_t*>(rest + at) = b;
            }
        }
}

}  // namespace

// ---------------------------------------------------------------- the tiles
//
// A tile is {first row, end row, start and end of its sequence}; rows outside
// every sequence make tiles of an empty sequence, whose outputs are zero, and
// if the starts are no starts at all (negative, falling, past the rows), all
// rows make tiles with end -1, whose outputs are NaN: no start that a caller
// passes leads a kernel out of its buffers.  `by_query` has the tiles with the
// most keys first, `by_key` those with the most queries, so that the longest
// run first and the short ones fill the gaps; entries that are left over hold
// no rows.  One workgroup, a wave a sequence and a lane a tile: a pass that
// counts tiles by their number in the sequence, a scan, a pass that places them.
// (The order within one count is free and changes no result.)  Also `pairs`, how
// often a tile of queries meets one of keys: those of rows in no sequence meet none.
#define BUCKETS 4096
#define BUILDERS 1024

__global__ void __launch_bounds__(BUILDERS)
packed_tiles_kernel(const int* __restrict__ starts, int B, int T, int max_tiles,
                    int4_t* __restrict__ by_query, int4_t* __restrict__ by_key,
                    float* __restrict__ pairs) {
    __shared__ int first[BUCKETS], fill_q[BUCKETS], fill_k[BUCKETS];
    __shared__ int total;
    __shared__ unsigned long long meet;   // whole, as its order is free
    const int tid = threadIdx.x;
    int shift = 0;
    while (((T / ROWS) >> shift) >= BUCKETS) ++shift;
    const int used = ((T / ROWS) >> shift) + 1;
    for (int i = tid; i < used; i += BUILDERS) first[i] = fill_q[i] = fill_k[i] = 0;
    if (tid == 0) meet = 0;
    // sequence 0 is the rows before the first one, B + 1 those behind the last;
    // a wave's lanes load 64 ranges at once, so that the loads overlap
    const int lane = tid & (WAVE - 1), wid = tid / WAVE;
    constexpr int WAVES = BUILDERS / WAVE;
    auto range = [&](int b, int& s, int& e) {
        s = b > 0 && b < B + 2 ? starts[b - 1] : 0;
        e = b <= B ? starts[b] : b < B + 2 ? T : 0;
    };
    const int mine = wid + lane * WAVES;
    int s0, e0;
    range(mine, s0, e0);   // all there are, up to 1022 sequences
    bool bad = s0 < 0 || e0 > T || e0 < s0;
    const auto meetings = [&](int b, int s, int e) {
        const unsigned long long n = ((unsigned)e - (unsigned)s + ROWS - 1) / ROWS;
        return b > 0 && b <= B ? n * (n + 1) / 2 : 0;
    };
    unsigned long long own = meetings(mine, s0, e0);
    for (int b = mine + BUILDERS; b < B + 2; b += BUILDERS) {
        int s, e;
        range(b, s, e);
        bad |= s < 0 || e > T || e < s;
        own += meetings(b, s, e);
    }
    const bool wrong = __syncthreads_or(bad);
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) own += __shfl_xor(own, off, WAVE);
    if (lane == 0 && !wrong) atomicAdd(&meet, own);
    auto each = [&](auto use) {
        for (int b0 = wid; b0 < B + 2; b0 += BUILDERS) {
            int s = s0, e = e0;
            if (b0 != wid) range(b0 + lane * WAVES, s, e);
            if (wrong) {
                s = 0;
                e = b0 + lane == 0 ? T : 0;
            }
            for (int j = 0; j < WAVE && b0 + j * WAVES < B + 2; ++j) {
                const int sj = __shfl(s, j, WAVE), ej = __shfl(e, j, WAVE);
                const int n = (ej - sj + ROWS - 1) / ROWS;
                for (int i = lane; i < n; i += WAVE) use(b0 + j * WAVES, sj, ej, n, i);
            }
        }
    };
    each([&](int, int, int, int, int i) { atomicAdd(&first[i >> shift], 1); });
    __syncthreads();
    // first[k] = number of tiles in buckets above k
    if (tid < WAVE) {
        int above = 0;
        for (int top = used - 1; top >= 0; top -= WAVE) {
            const int k = top - tid;
            const int n = k >= 0 ? first[k] : 0;
            int sum = n;
#pragma unroll
            for (int off = 1; off < WAVE; off <<= 1) {
                const int v = __shfl_up(sum, off, WAVE);
                if (tid >= off) sum += v;
            }
            if (k >= 0) first[k] = above + sum - n;
            above += __shfl(sum, WAVE - 1, WAVE);
        }
        if (tid == 0) {
            total = above;
            *pairs = (float)meet;
        }
    }
    __syncthreads();
    each([&](int b, int s, int e, int n, int i) {
        const bool real = !wrong && b > 0 && b <= B;
        const int r0 = s + i * ROWS;
        const int4_t t = {r0, min(r0 + ROWS, e), real ? s : r0, real ? e : wrong ? -1 : r0};
        const int kq = i >> shift, kk = (n - 1 - i) >> shift;
        const int at_q = first[kq] + atomicAdd(&fill_q[kq], 1);
        const int at_k = first[kk] + atomicAdd(&fill_k[kk], 1);
        if (at_q < max_tiles) by_query[at_q] = t;
        if (at_k < max_tiles) by_key[at_k] = t;
    });
    for (int i = total + tid; i < max_tiles; i += BUILDERS)
        by_query[i] = by_key[i] = int4_t{0, 0, 0, 0};
}

// op(x, y, ...) of the wave's lanes, with 0 for none
template <typename Op>
DEVINL int wave_fold(int x, Op op) {
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));   // row_shr 1, 2,
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));   // 4, 8: within
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));   // each 16 lanes
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));   // row_bcast 15, 31
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, WAVE - 1);
}

// Entry p of that table by query, found by every wave for itself, a lane a
// sequence, for up to PACKED_FEW sequences.  How many tiles are the i-th or later
// of their sequence falls with i: a search for the i where it passes p.  (Also
// entry p by key, and `pairs`.)
DEVINL int4_t find_tile(const int* __restrict__ starts, int B, int T, int p, int4_t& by_key,
                        float& pairs) {
    const int b = threadIdx.x & (WAVE - 1);
    int s = b > 0 && b < B + 2 ? starts[b - 1] : 0;
    int e = b <= B ? starts[b] : b < B + 2 ? T : 0;
    const bool wrong = __any(s < 0 || e > T || e < s);
    if (wrong) {
        s = 0;
        e = b == 0 ? T : 0;
    }
    const int n = (e - s + ROWS - 1) / ROWS;
    const bool in = !wrong && b > 0 && b <= B;
    pairs = in ? 0.5f * n * (n + 1.f) : 0.f;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) pairs += __shfl_xor(pairs, off, WAVE);
    const auto sum = [](int x, int y) { return x + y; };
    by_key = int4_t{0, 0, 0, 0};
    if (wave_fold(n, sum) <= p) return by_key;
    int i = 0, past = wave_fold(n, [](int x, int y) { return max(x, y); });
    int before = 0;   // tiles that are the past-th or later
    while (past - i > 1) {
        const int mid = (i + past) / 2, later = wave_fold(max(n - mid, 0), sum);
        if (later > p) {
            i = mid;
        } else {
            past = mid;
            before = later;
        }
    }
    const unsigned long have = __ballot(n > i);
    const int rank = __popcll(have & ((1ul << b) - 1));
    const int seq = __ffsll(__ballot(n > i && rank == p - before)) - 1;
    s = __builtin_amdgcn_readlane(s, seq);
    e = __builtin_amdgcn_readlane(e, seq);
    const int last = __builtin_amdgcn_readlane(n, seq) - 1;
    const bool real = !wrong && seq > 0 && seq <= B;
    const auto tile = [&](int i) {
        const int r0 = s + i * ROWS;
        return int4_t{r0, min(r0 + ROWS, e), real ? s : r0, real ? e : wrong ? -1 : r0};
    };
    by_key = tile(last - i);
    return tile(i);
}

// Which tile (or half tile) and head workgroup i of the forward and dq kernels
// takes.  Workgroups go round the 8 XCDs in turn, and each XCD has an L2 of its
// own, so all heads of a group take a tile one after the other on one XCD: its
// keys come there once.  With 8n kv heads an XCD has kv heads of its own; with
// 1, 2 or 4, 8/Hk XCDs share one and take every 8/Hk-th tile of it.
struct Place { int tile, hk, h; };
DEVINL Place place_of(int i, int Hq, int Hk) {
    const int group = Hq / Hk;
    if (8 % Hk == 0) {
        const int share = 8 / Hk, lane = i % 8, turn = i / 8, hk = lane % Hk;
        return {turn / group * share + lane / Hk, hk, hk * group + turn % group};
    }
    const int hk = i % Hk;
    return {i / Hq, hk, hk * group + i % Hq / Hk};
}

// ------------------------------------------------------------------ forward
//
// A workgroup takes a tile of 128 rows of one head, a wave 32 of the rows.  64
// keys at a time stand in LDS, the next ones are on their way there meanwhile.
// With two TEAMS it takes half a tile, and each team half of the keys, whose
// sums are joined at the end: for grids that leave CUs idle, where a wave's own
// chain of steps is what takes the time.
//
// Bound by the SIMDs: a wave's MFMA (16 a block of 32 keys at D 128, 15 ns each)
// and the softmax's VALU work (3.4 ns an exp2, 1 ns an add) hardly hide beneath each
// other, other waves' neither.  By the counters, of all SIMDs' cycles: 8192 rows, D
// 128: MFMA 56 %, VALU 42 %.  The policy's batch, D 64: MFMA 31 %, VALU 52 %, and
// CUs are empty for 24 % of the time (starts, ends, short sequences' first loads;
// also a tenth of its blocks are of waves whose rows lie past the sequence).  A wave keeps 32 rows because each fragment
// of K and V from LDS then serves a product of 32 columns, and 128 registers of
// accumulators and queries still leave two workgroups a CU.  Two of them overlap
// each other's softmax and products better than one with longer tiles (two
// blocks at a time in one wave: 631 against 590 us).  Without loads and barriers
// 8192 rows still took 477 us of 558; the rest is these.  8192 rows, 32/8 heads of
// 128: 0.49 to 0.55 ms by card and clock, 1.0 to 1.12 PFLOP/s; 32768 rows in sequences
// of 64 to 1536, 8/4 heads of 64: 55 to 60 us, 0.6 to 0.65 PFLOP/s.
template <int D, int TEAMS, bool SAVE>
__global__ void __launch_bounds__(256, D == 128 ? 2 : 4)
packed_attn_fwd_kernel(const PackedArgs a) {
    const int T = a.T, Hq = a.Hq, Hk = a.Hk;
    int4_t* tiles = (int4_t*)a.tiles;
    const Place place = place_of(blockIdx.x, Hq, Hk);
    const int hk = place.hk, h = place.h, at_tile = place.tile / TEAMS;
    if (at_tile >= a.max_tiles) return;
    int4_t tile;
    if (a.search) {
        int4_t by_key;
        float pairs;
        tile = find_tile(a.starts, a.B, T, at_tile, by_key, pairs);
        // the table for the backward pass
        if (SAVE && h == 0 && place.tile % TEAMS == 0 && threadIdx.x == 0) {
            tiles[at_tile] = tile;
            tiles[a.max_tiles + at_tile] = by_key;
            if (at_tile == 0) *(float*)(tiles + 2 * (long)a.max_tiles) = pairs;
        }
    } else {
        tile = tiles[at_tile];
    }
    const int row0 = tile[0] + place.tile % TEAMS * (ROWS / TEAMS);
    const int row1 = min(tile[1], row0 + ROWS / TEAMS), seq0 = tile[2], seq1 = tile[3];
    if (row0 >= row1) return;
    const bool real = seq1 > seq0;
    const int kv0 = seq0, kv1 = real ? row1 : seq0;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int hi = lane >> 5;
    constexpr int SETS = 4 / TEAMS;   // of 32 rows
    const int team = wid / SETS;
    const int wrow = row0 + wid % SETS * 32;
    const int row = wrow + (lane & 31);
    const bool mine = row < row1;
    const float c2 = __uint_as_float(__builtin_amdgcn_readfirstlane(
        __float_as_uint(a.scale * LOG2E)));

    constexpr int N = D / 16, AHEAD = 4;   // products of a kind, fragments read ahead
    // two tiles of keys, two of values
    constexpr int TILE = 64 * D * 2;
    __shared__ __attribute__((aligned(256))) char lds[4 * TILE];
    const Lane<D, true> lanes(lane);

    bf16x8_t qf[D / 16];
    load_row<D>(qf, a.q + row * a.qt + h * a.qh, mine, hi);
    f32x16_t acc[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db) acc[db] = zero16();
    float m = -INFINITY, l = 0.f;
    const ushort_t *k = a.k + hk * a.kh, *v = a.v + hk * a.vh;
    const Mover<D, 64, 256> mk(a.kt), mv(a.vt);
    const int steps = (kv1 - kv0 + 63) / 64;
    const char *knext = mk.at(k, kv0), *vnext = mv.at(v, kv0);
    auto fetch = [&](int it) {
        mk.move(knext, kv1 - 1 - (kv0 + it * 64), lds + (it & 1) * TILE);
        mv.move(vnext, kv1 - 1 - (kv0 + it * 64), lds + (2 + (it & 1)) * TILE);
        knext += 64 * mk.pitch;
        vnext += 64 * mv.pitch;
    };
    if (steps > 0) fetch(0);
    settle(qf);
    arrived();
    __syncthreads();
    const int wave_end = min(wrow + 32, row1);   // keys this wave's rows reach
    auto step = [&](auto buf, int it) {
        // into the tiles that were last read before the barrier of the step before
        if (it + 1 < steps) fetch(it + 1);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int key0 = kv0 + it * 64 + sub * 32;
            if (key0 >= wave_end || (TEAMS > 1 && sub != team)) continue;
            // a product each: N fragments of K, then N of V^T
            char* const tile = lds + buf * TILE + sub * (TILE / 2);
            auto fragment = [&](int i) {
                return i < N ? rows_frag(tile, lanes, i)
                             : cols_frag<D>(tile + 2 * TILE + (i - N) / (D / 32) * (TILE / 4),
                                            lanes, (i - N) % (D / 32));
            };
            bf16x8_t f[AHEAD];
            auto next = [&](int i) {
                if (i + AHEAD < 2 * N) f[i % AHEAD] = fragment(i + AHEAD);
                in_order<D>();
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) f[i] = fragment(i);
            in_order<D>();
            f32x16_t s = zero16();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s = mfma(f[i % AHEAD], qf[i], s);
                next(i);
            }
            if (key0 + 31 > wrow) {   // not every key open to every row
                const int open = seldom(row - key0 - 4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (crow(r, 0) > open) s[r] = -INFINITY;
            }
            f32x16_t p;
            float sum;
            auto weigh = [&](float base) {
                sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, -base));
                    sum += p[r];
                }
            };
            weigh(m);
            // P is taken by the maximum so far: as long as no half row sums to more
            // than 2^13 that costs no bits, and the block's own maximum is not
            // needed.  (At first m is -inf, and the sum infinite or NaN.)
            if (!__all(sum <= 8192.f)) {
                float top = s[0];
#pragma unroll
                for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
                const float to = fmaxf(m, both_max(top) * c2);
                const float base = to == -INFINITY ? 0.f : to;
                const float f = __builtin_amdgcn_exp2f(m - base);
                m = to;
                l *= f;
#pragma unroll
                for (int db = 0; db < D / 32; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[db][r] *= f;
                weigh(base);
            }
            l += sum;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                acc[i % (D / 32)] = mfma(f[(N + i) % AHEAD], pack8(p, i / (N / 2)),
                                         acc[i % (D / 32)]);
                next(N + i);
            }
        }
        arrived();
        __syncthreads();
    };
    for (int it = 0; it < steps; it += 2) {
        step(std::integral_constant<int, 0>{}, it);
        if (it + 1 < steps) step(std::integral_constant<int, 1>{}, it + 1);
    }
    if (TEAMS > 1) {
        // the second team's rows to the first
        float* join = reinterpret_cast<float*>(lds) + wid % SETS * (D / 2 + 2) * 64 + lane;
        if (team) {
            join[0] = m;
            join[64] = l;
#pragma unroll
            for (int i = 0; i < D / 2; ++i) join[(2 + i) * 64] = acc[i / 16][i % 16];
        }
        __syncthreads();
        if (team) return;
        const float m2 = join[0], to = fmaxf(m, m2), base = to == -INFINITY ? 0.f : to;
        const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
        m = to;
        l = l * f + join[64] * f2;
#pragma unroll
        for (int i = 0; i < D / 2; ++i)
            acc[i / 16][i % 16] = acc[i / 16][i % 16] * f + join[(2 + i) * 64] * f2;
    }
    l = both_sum(l);
    const long to = ((long)row * Hq + h) * D;
    store_row<D>(acc, seq1 < 0 ? NAN : real ? 1.f / l : 0.f, a.out + to, hi,
                 SAVE ? a.out_lo + to : nullptr, mine);
    if (SAVE && mine && hi == 0) a.lse[(long)h * T + row] = m + __builtin_amdgcn_logf(l);
}

// ----------------------------------------------------------------------- dq
//
// The forward kernel's split.  Also writes -delta for the kernel below.  24 MFMA
// a block of 32 keys at D 128 and less VALU work than forward (no maximum): MFMA are
// busy 54 % of the time and VALU 32 %, with D 64 35 and 49 %.  4096 + 2500 + 1000 + 596
// rows, 32/8 heads of 128: 0.28 to 0.32 ms, 0.94 to 1.07 PFLOP/s; 32768 rows of the
// policy: 76 to 85 us, 0.64 to 0.71 PFLOP/s.
template <int D, int TEAMS>
__global__ void __launch_bounds__(256, D == 128 ? 2 : 4)
packed_attn_dq_kernel(const PackedArgs a) {
    const int T = a.T, Hq = a.Hq, Hk = a.Hk;
    const int4_t* tiles = (const int4_t*)a.tiles;
    const Place place = place_of(blockIdx.x, Hq, Hk);
    const int hk = place.hk, h = place.h, at_tile = place.tile / TEAMS;
    if (a.parts > 1 && threadIdx.x < 2) {   // for the kernel below
        const unsigned i = 2 * blockIdx.x + threadIdx.x;
        if (i < (unsigned)a.counters) a.counts[i] = 0;
    }
    if (at_tile >= a.max_tiles) return;
    const int4_t tile = tiles[at_tile];
    const int row0 = tile[0] + place.tile % TEAMS * (ROWS / TEAMS);
    const int row1 = min(tile[1], row0 + ROWS / TEAMS), seq0 = tile[2], seq1 = tile[3];
    if (row0 >= row1) return;
    const bool real = seq1 > seq0;
    const int kv0 = seq0, kv1 = real ? row1 : seq0;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int hi = lane >> 5;
    constexpr int SETS = 4 / TEAMS;   // of 32 rows
    const int team = wid / SETS;
    const int wrow = row0 + wid % SETS * 32;
    const int row = wrow + (lane & 31);
    const bool mine = row < row1;
    const float c2 = __uint_as_float(__builtin_amdgcn_readfirstlane(
        __float_as_uint(a.scale * LOG2E)));

    constexpr int N = D / 16, AHEAD = D == 128 ? 4 : 1;   // products of a kind, fragments read ahead
    constexpr int TILE = 64 * D * 2;
    __shared__ __attribute__((aligned(256))) char lds[4 * TILE];
    constexpr bool KEPT = D == 128;
    const Lane<D, KEPT> lanes(lane);

    const ushort_t *k = a.k + hk * a.kh, *v = a.v + hk * a.vh;
    const Mover<D, 64, 256> mk(a.kt), mv(a.vt);
    const int steps = (kv1 - kv0 + 63) / 64;
    const char *knext = mk.at(k, kv0), *vnext = mv.at(v, kv0);
    auto fetch = [&](int it) {
        mk.move(knext, kv1 - 1 - (kv0 + it * 64), lds + (it & 1) * TILE);
        mv.move(vnext, kv1 - 1 - (kv0 + it * 64), lds + (2 + (it & 1)) * TILE);
        knext += 64 * mk.pitch;
        vnext += 64 * mv.pitch;
    };
    if (steps > 0) fetch(0);
    bf16x8_t qf[D / 16], of[D / 16];
    load_row<D>(qf, a.q + row * a.qt + h * a.qh, mine, hi);
    load_row<D>(of, a.dout + row * a.ot + h * a.oh, mine, hi);
    float ls = mine ? a.lse[(long)h * T + row] : 0.f;
    float dl = 0.f;
    {
        bf16x8_t o[D / 16], rest[D / 16];
        load_row<D>(o, a.out + ((long)row * Hq + h) * D, mine, hi);
        load_row<D>(rest, a.out_lo + ((long)row * Hq + h) * D, mine, hi);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                dl = fmaf((float)of[s][j], (float)o[s][j] + (float)rest[s][j], dl);
        dl = both_sum(dl);
    }
    settle(qf);
    settle(of);
    asm volatile("" : "+v"(ls));
    f32x16_t acc[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db) acc[db] = zero16();
    const int wave_end = min(wrow + 32, row1);
    // One pass over the keys.  Of P and dP, `use` makes what the pass is for, with
    // COUNT fragments of each block read in all.
    auto sweep = [&](auto count, auto use) {
        constexpr int COUNT = decltype(count)::value;
        // dP is summed onto -delta, for which D 64 has no 16 registers to spare
        constexpr bool LESS = D == 128 && COUNT == 3 * N;
        f32x16_t less;
#pragma unroll
        for (int r = 0; r < 16; ++r) less[r] = -dl;
        if (LESS) asm volatile("" : "+v"(less));   // once, not every block
        arrived();   // the first tiles
        __syncthreads();
        auto step = [&](auto buf, int it) {
            if (it + 1 < steps) fetch(it + 1);
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int key0 = kv0 + it * 64 + sub * 32;
                if (key0 >= wave_end || (TEAMS > 1 && sub != team)) continue;
                // a product each: N fragments of K, N of V, N of K^T for `use`
                const int off = buf * TILE + sub * (TILE / 2);
                const Lane<D, KEPT> at = lanes.fresh(off);
                char* const tile = KEPT ? lds + off : lds;
                auto fragment = [&](int i) {
                    return i < N       ? rows_frag(tile, at, i)
                           : i < 2 * N ? rows_frag(tile + 2 * TILE, at, i - N)
                                       : cols_frag<D>(tile + (i - 2 * N) / (D / 32) * (TILE / 4),
                                                      at, (i - 2 * N) % (D / 32));
                };
                bf16x8_t f[AHEAD];
                auto next = [&](int i) {
                    if (i + AHEAD < COUNT) f[i % AHEAD] = fragment(i + AHEAD);
                    in_order<D>();
                };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) f[i] = fragment(i);
                in_order<D>();
                f32x16_t s = zero16(), dp = LESS ? less : zero16();
                auto weigh = [&](int r) {
                    s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, -ls));
                };
                // with D 128 the exp of S goes beneath the products of dP
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s = mfma(f[i % AHEAD], qf[i], s);
                    next(i);
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    dp = mfma(f[(N + i) % AHEAD], of[i], dp);
                    if (D == 128)
#pragma unroll
                        for (int r = beneath(i, N); r < beneath(i + 1, N); ++r) weigh(r);
                    next(N + i);
                }
                if (D == 64)
#pragma unroll
                    for (int r = 0; r < 16; ++r) weigh(r);
                if (key0 + 31 > wrow) {   // not every key open to every row
                    const int open = seldom(row - key0 - 4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (crow(r, 0) > open) s[r] = 0.f;
                }
                use(s, dp, f, next);
            }
            arrived();
            __syncthreads();
        };
        for (int it = 0; it < steps; it += KEPT ? 2 : 1) {
            if (KEPT) {
                step(std::integral_constant<int, 0>{}, it);
                if (it + 1 < steps) step(std::integral_constant<int, 1>{}, it + 1);
            } else {
                step(it & 1, it);
            }
        }
    };
    float* join = reinterpret_cast<float*>(lds) + wid % SETS * (D / 2) * 64 + lane;
    if (tile[0] == seq0) {
        float sum = 0.f;
        sweep(std::integral_constant<int, 2 * N>{}, [&](f32x16_t& p, f32x16_t& dp, auto&, auto&) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sum = fmaf(p[r], dp[r], sum);
        });
        if (TEAMS > 1) {
            // each team's sum to the other
            join[team * SETS * (D / 2) * 64] = sum;
            __syncthreads();
            sum += join[(1 - team) * SETS * (D / 2) * 64];
            __syncthreads();
        }
        dl = both_sum(sum);
        knext = mk.at(k, kv0);
        vnext = mv.at(v, kv0);
        if (steps > 0) fetch(0);
    }
    if (mine && hi == 0 && team == 0) a.delta[(long)h * T + row] = -dl;
    sweep(std::integral_constant<int, 3 * N>{}, [&](f32x16_t& p, f32x16_t& dp, auto& f, auto& next) {
#pragma unroll
        for (int r = 0; r < 8; ++r) p[r] *= D == 128 ? dp[r] : dp[r] - dl;
        bf16x8_t df = pack8(p, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i == N / 2) df = pack8(p, 1);
            acc[i % (D / 32)] = mfma(f[(2 * N + i) % AHEAD], df, acc[i % (D / 32)]);
            if (i < N / 2)
#pragma unroll
                for (int r = 8 + i * (16 / N); r < 8 + (i + 1) * (16 / N); ++r)
                    p[r] *= D == 128 ? dp[r] : dp[r] - dl;
            next(2 * N + i);
        }
    });
    if (TEAMS > 1) {
        if (team)
#pragma unroll
            for (int i = 0; i < D / 2; ++i) join[i * 64] = acc[i / 16][i % 16];
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int i = 0; i < D / 2; ++i) acc[i / 16][i % 16] += join[i * 64];
    }
    store_row<D>(acc, seq1 < 0 ? NAN : a.scale, a.dq + ((long)row * Hq + h) * D, hi, nullptr, mine);
}

// ------------------------------------------------------------------- dk, dv
//
// A workgroup takes KS sets of 32 keys of one kv head (a tile or a half of it);
// the queries of all the group's heads that see them pass through LDS, QB at a
// time.  A wave keeps k and v of one set in registers; KS waves share the keys,
// two teams of them the queries, and their sums are joined at the end.
//
// These workgroups are few and of unequal length (the first keys are seen by all
// queries), and the longest can take far longer than the card's share of the
// work.  So the queries of a long one are split in up to `parts` workgroups.
// Each leaves its sums in memory and counts itself; the last to come adds all
// sums in their order, so the same inputs give the same bits, and nobody waits.
// Sums and count go past the caches (relaxed atomics of agent scope): a fence
// would write back and drop an XCD's whole L2, which made everything slower (1.06
// ms instead of 0.81).  So the order of sums before count rests on the hardware, not
// on the language's memory model: s_waitcnt vmcnt(0) ends when every write-through
// store of the wave has reached memory, all waves wait for that and meet at the
// barrier, and only then one thread counts.  What keeps the compiler from moving the
// stores past that wait is that it is volatile asm with a memory clobber; on the
// other side the loads stand behind the barrier that follows the count.  The parts
// are the outer order of the grid, as the many that are not there would else leave
// every other CU idle.
//
// 32 MFMA a block of 32 x 32 at D 128, and as many 1 KB fragments from LDS, each
// read for one product.  LDS is busy 27 % of the time, the matrix cores 42 % and
// VALU 27 %, none of which overlap in full, and a wave has no registers left to read
// far ahead (256; 64 keys a wave, which would halve the
// reads, spilled: 761 against 510 us).  At D 128 one workgroup of 8 waves has all
// of LDS, so that a tile of 128 queries serves 128 keys; at D 64 three buffers of
// 64 queries keep two tiles on their way.  4096 + 2500 + 1000 + 596 rows, 32/8
// heads of 128: 0.42 to 0.51 ms, 0.79 to 0.95 PFLOP/s (0.51 unsplit where that was
// 0.46); 32768 rows of the policy: 97 to 106 us, 0.68 to 0.75 PFLOP/s.
//
// WHOLE: no workgroup is split that lacks some of its keys.  More than WORTH steps
// are more than WORTH / group turns of QB queries, so with groups of up to 8 heads
// at least the tile's 128 rows lie between its first key and the sequence's end.
template <int D, int KS, int QB, int NBUF, bool WHOLE>
__global__ void __launch_bounds__(KS * 128, D == 128 ? 2 : 3)
packed_attn_dkv_kernel(const PackedArgs a) {
    const int T = a.T, Hq = a.Hq, Hk = a.Hk;
    const int4_t* tiles = (const int4_t*)a.tiles + a.max_tiles;
    const float pairs = *(const float*)(tiles + a.max_tiles);
    static_assert(QB == KS * 32 && QB == packed_keys(D), "as many queries as keys");
    constexpr int TEAMS = 2, BITS = 4 / KS, SLOTS = packed_slots(D), WORTH = packed_worth(D);
    const int hk = blockIdx.x % Hk;
    const int group = Hq / Hk;
    // first the last parts, which few tiles have, and those few the first ones
    const int bits = a.max_tiles * BITS;
    const int part = a.parts - 1 - blockIdx.x / Hk / bits;
    const int bit = blockIdx.x / Hk % bits;
    const int at_tile = bit / BITS;
    const int4_t tile = tiles[at_tile];
    // The first half of a tile is seen by more queries, and the second may be
    // empty.  Workgroups go round the XCDs, and round the engines of one, in a
    // fixed order: which half comes first changes from tile to tile so that no
    // period of two, four or eight workgroups has all of a kind.
    const int row0 = tile[0] + (bit + (BITS > 1 ? __popc(at_tile) : 0)) % BITS * (KS * 32);
    const int row1 = tile[1], seq0 = tile[2], seq1 = tile[3];
    if (row0 >= row1) return;
    const bool real = seq1 > seq0;
    // Steps of QB of one head's queries that see the keys, and the steps that come
    // to each slot if all are shared out: what would take WORTH steps longer is
    // split (where all workgroups run at once, already over three quarters of it).
    const int turns = (seq1 - row0 + QB - 1) / QB, all = real ? turns * group : 0;
    const float share =
        pairs * ((ROWS / QB) * (ROWS / QB) * Hq) / SLOTS * (a.parts > 2 ? 0.75f : 1.f);
    const int parts = __builtin_amdgcn_readfirstlane(
        all > share + WORTH ? min(a.parts, (int)ceilf(all / fmaxf(share, WORTH / 2.f))) : 1);
    if (part >= parts) return;
    const int step0 = (int)((long)all * part / parts);
    const int steps = (int)((long)all * (part + 1) / parts) - step0;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int hi = lane >> 5;
    const int team = wid / KS;
    const int wkey = row0 + wid % KS * 32;
    const int key = wkey + (lane & 31);
    const bool mine = key < row1;
    const float c2 = a.scale * LOG2E;

    // NBUF tiles of queries, as many of their outputs' gradients, and each row's
    // log-sum and negated delta
    constexpr int TILE = QB * D * 2;
    struct __attribute__((aligned(256))) Lds {
        char x[2 * NBUF * TILE];
        float ls[NBUF][QB], dl[NBUF][QB];
    };
    __shared__ Lds lds;
    char* const ql = lds.x;
    char* const ol = lds.x + NBUF * TILE;
    const Lane<D, false> lanes(lane);

    bf16x8_t kf[D / 16], vf[D / 16];
    f32x16_t ak[D / 32], av[D / 32];
    load_row<D>(kf, a.k + key * a.kt + hk * a.kh, mine, hi);
    load_row<D>(vf, a.v + key * a.vt + hk * a.vh, mine, hi);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) ak[db] = av[db] = zero16();

    const Mover<D, QB, KS * TEAMS * 64> mq(a.qt), mo(a.ot);
    // each wave also moves 64 rows' log-sums or deltas (where there are more
    // waves than these, two move the same)
    static_assert(QB % 64 == 0 && KS * TEAMS % (QB / 32) == 0, "by wave");
    const int rows64 = wid % (QB / 32) / 2;
    const bool sums = wid % 2 == 0;
    constexpr int AHEAD = NBUF - 1, LEFT = (NBUF - 2) * (2 * mq.LOADS + 1);
    // what is fetched next
    const int start = real ? row0 + step0 % turns * QB : row0;
    int h = hk * group + (real ? step0 / turns : 0), r0 = start;
    const float* const rows = sums ? a.lse : a.delta;
    const char *qnext, *onext;
    const float* snext;
    auto begin = [&] {
        qnext = mq.at(a.q + h * a.qh, r0);
        onext = mo.at(a.dout + h * a.oh, r0);
        snext = rows + (long)h * T + r0;
    };
    begin();
    auto next = [&](int buf) {
        const int last = seq1 - 1 - r0;
        mq.move(qnext, last, ql + buf * TILE);
        mo.move(onext, last, ol + buf * TILE);
        move64(snext, min(rows64 * 64 + lane, last),
               (sums ? lds.ls[buf] : lds.dl[buf]) + rows64 * 64);
        r0 += QB;
        qnext += QB * mq.pitch;
        onext += QB * mo.pitch;
        snext += QB;
        if (r0 >= seq1) {
            r0 = row0;
            ++h;
            begin();
        }
    };
#pragma unroll
    for (int it = 0; it < AHEAD; ++it)
        if (it < steps) next(it);
    settle(kf);
    settle(vf);
    if (steps >= AHEAD) arrived<LEFT>();
    else arrived<0>();
    __syncthreads();
    int now = start;   // first row of the step
    for (int it = 0, buf = 0; it < steps; ++it, buf = buf + 1 < NBUF ? buf + 1 : 0) {
        const bool more = it + AHEAD < steps;
        if (more) next(buf ? buf - 1 : NBUF - 1);
#pragma unroll 1
        for (int sub = 0; sub < QB / 32 / TEAMS; ++sub) {
            const int in = (team * (QB / 32 / TEAMS) + sub) * 32;   // first row in the tile
            const int first = now + in;
            // queries all before the wave's keys, or past the sequence
            if (first + 31 < wkey || first >= seq1) continue;
            const Lane<D, false> at = lanes.fresh(buf * TILE + in * (D * 2));
            f32x16_t s = zero16(), dp;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
                s = mfma(rows_frag(ql, at, d), kf[d], s);
            // dP - delta, summed onto the deltas
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4_t dl = *reinterpret_cast<const float4_t*>(
                    &lds.dl[buf][in + 8 * g + 4 * hi]);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[4 * g + j] = dl[j];
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
                dp = mfma(rows_frag(ol, at, d), vf[d], dp);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4_t ls = *reinterpret_cast<const float4_t*>(
                    &lds.ls[buf][in + 8 * g + 4 * hi]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], c2, -ls[j]));
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] *= s[r];
            // some do not see some, or are past the sequence
            if (first < wkey + 31 || first + 31 >= seq1) {
                const int lo = seldom(key - first - 4 * hi), hi_ = seq1 - first - 4 * hi;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (crow(r, 0) < lo || crow(r, 0) >= hi_) s[r] = dp[r] = 0.f;
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const bf16x8_t pf = pack8(s, ks);
#pragma unroll
                for (int db = 0; db < D / 32; ++db)
                    av[db] = mfma(cols_frag<D>(ol + ks * (32 * D), at, db), pf,
                                  av[db]);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const bf16x8_t df = pack8(dp, ks);
#pragma unroll
                for (int db = 0; db < D / 32; ++db)
                    ak[db] = mfma(cols_frag<D>(ql + ks * (32 * D), at, db), df,
                                  ak[db]);
            }
        }
        now += QB;
        if (now >= seq1) now = row0;
        if (more) arrived<LEFT>();
        else arrived<0>();
        __syncthreads();
    }
    // dv to the first team, then dk to the second
    auto joined = [&](f32x16_t (&x)[D / 32], int to) {
        float* join = reinterpret_cast<float*>(lds.x) + wid % KS * 32 * D + lane;
        static_assert(KS * 32 * D * 4 <= 2 * NBUF * TILE, "fits the tiles");
        if (team != to)
#pragma unroll
            for (int i = 0; i < D / 2; ++i) join[i * 64] = x[i / 16][i % 16];
        __syncthreads();
        if (team == to)
#pragma unroll
            for (int i = 0; i < D / 2; ++i) x[i / 16][i % 16] += join[i * 64];
    };
    joined(av, 0);
    __syncthreads();
    joined(ak, 1);
    if (team == 1)   // from here on av is dv with team 0 and dk with team 1
#pragma unroll
        for (int db = 0; db < D / 32; ++db) av[db] = ak[db];
    if (parts > 1) {
        // The last workgroup of the parts adds them all, in their order.  A part's
        // sums are laid out by the rows of dk and dv that they are for, a wave's rows
        // one after the other element by element: no more memory than those rows.
        union Two { float f[2]; unsigned long u; };
        const long slot = (long)bit * Hk + hk;
        // (Where the rows are known the offsets are constants: 8/4 heads of 64, 1023
        // rows and some short sequences, 19.0 us; as variables 19.9.)
        const int wave_rows =   // below 1 none is `mine`
            WHOLE ? 32 : __builtin_amdgcn_readfirstlane(min(32, row1 - wkey));
        // use(pair i, where it is)
        auto sums = [&](int part, auto use) {
            unsigned long* const at =
                reinterpret_cast<unsigned long*>(
                    a.sums + ((((long)part * Hk + hk) * 2 + team) * T + wkey) * D) +
                hi * wave_rows + (lane & 31);
            if (WHOLE || mine)
#pragma unroll
                for (int i = 0; i < D / 4; ++i) use(i, at + i * 2 * wave_rows);
        };
        sums(part, [&](int i, unsigned long* at) {
            __hip_atomic_store(at, Two{{av[i / 8][i % 8 * 2], av[i / 8][i % 8 * 2 + 1]}}.u,
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        });
        arrived();
        __syncthreads();
        int& before = reinterpret_cast<int*>(lds.x)[0];
        if (threadIdx.x == 0)
            before = __hip_atomic_fetch_add(a.counts + slot, 1, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (before != parts - 1) return;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) av[db] = zero16();
        for (int p = 0; p < parts; ++p)
            sums(p, [&](int i, unsigned long* at) {
                Two v;
                v.u = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                av[i / 8][i % 8 * 2] += v.f[0];
                av[i / 8][i % 8 * 2 + 1] += v.f[1];
            });
    }
    const long to = ((long)key * Hk + hk) * D;
    const float factor = seq1 < 0 ? NAN : team ? a.scale : 1.f;
    store_row<D>(av, factor, (team ? a.dk : a.dv) + to, hi, nullptr, mine);
}

// ---------------------------------------------------------------- launchers
// Each returns the launch's hipError_t.

extern "C" int launch_packed_tiles(const PackedArgs* a, void* stream) {
    int4_t* tiles = (int4_t*)a->tiles;
    hipLaunchKernelGGL(packed_tiles_kernel, dim3(1), dim3(BUILDERS), 0, (hipStream_t)stream,
                       a->starts, a->B, a->T, a->max_tiles, tiles, tiles + a->max_tiles,
                       (float*)(tiles + 2 * (long)a->max_tiles));
    return (int)hipGetLastError();
}

namespace {

// Workgroups that place_of() gives each of `tiles` tiles and every head
dim3 grid_of(const PackedArgs* a, int tiles) {
    const int share = 8 % a->Hk ? 1 : 8 / a->Hk;
    return dim3((unsigned)((tiles + share - 1) / share * share) * a->Hq);
}

template <int D, int TEAMS>
void fwd(const PackedArgs* a, hipStream_t st) {
    const dim3 grid = grid_of(a, a->max_tiles * TEAMS), block(256);
    if (a->lse)
        hipLaunchKernelGGL((packed_attn_fwd_kernel<D, TEAMS, true>), grid, block, 0, st, *a);
    else hipLaunchKernelGGL((packed_attn_fwd_kernel<D, TEAMS, false>), grid, block, 0, st, *a);
}

template <int D, int TEAMS>
void dq_(const PackedArgs* a, hipStream_t st) {
    hipLaunchKernelGGL((packed_attn_dq_kernel<D, TEAMS>),
                       grid_of(a, a->max_tiles * TEAMS), dim3(256), 0, st, *a);
}

template <int D, int KS, int QB, int NBUF>
void dkv(const PackedArgs* a, hipStream_t st) {
    static_assert(packed_worth(D) / 8 * QB >= ROWS, "WHOLE with up to 8 heads a group");
    const dim3 grid((unsigned)a->max_tiles * a->Hk * (4 / KS) * a->parts), block(KS * 128);
    if (a->Hq / a->Hk <= 8)
        hipLaunchKernelGGL((packed_attn_dkv_kernel<D, KS, QB, NBUF, true>), grid, block, 0, st, *a);
    else hipLaunchKernelGGL((packed_attn_dkv_kernel<D, KS, QB, NBUF, false>), grid, block, 0, st, *a);
}

// Whether the usual split leaves CUs with a workgroup or two less than fit: then
// two teams of waves take a tile.  With and without (us; 8/4 heads of 64, 32/8 of
// 128):
//   workgroups           forward     dq
//   88   1024, 8/4       14.5 19.2   17.0 22.1
//   328  3 x 1536, 8/4   26.4 32.5   31.4 37.5
//   448  6 x 1024, 8/4   23.4 27.5   28.3 32.5
//   736  1916, 32/8      33.6 33.4   47.4 43.7
bool sparse(const PackedArgs* a) { return a->max_tiles * a->Hq <= 512; }

}  // namespace

extern "C" int launch_packed_attn_fwd(const PackedArgs* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const bool few = sparse(a);
    if (a->D == 128) few ? fwd<128, 2>(a, st) : fwd<128, 1>(a, st);
    else few ? fwd<64, 2>(a, st) : fwd<64, 1>(a, st);
    return (int)hipGetLastError();
}

extern "C" int launch_packed_attn_dq(const PackedArgs* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const bool few = sparse(a);
    if (a->D == 128) few ? dq_<128, 2>(a, st) : dq_<128, 1>(a, st);
    else few ? dq_<64, 2>(a, st) : dq_<64, 1>(a, st);
    return (int)hipGetLastError();
}

extern "C" int launch_packed_attn_dkv(const PackedArgs* a, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    if (a->D == 128) dkv<128, 4, 128, 2>(a, st);
    else dkv<64, 2, 64, 3>(a, st);
    return (int)hipGetLastError();
}
