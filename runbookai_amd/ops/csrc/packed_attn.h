// What the packed-attention kernels and their bindings share.
#pragma once

#define PACKED_ROWS 128   // rows of a tile, of queries or of keys
#define PACKED_FEW 62     // sequences that a wave can look through by itself

// Passed by value as the kernels' argument.  The strides are in elements: of q
// from token to token (qt) and from head to head (qh), and so on; the last
// dimension is dense, all else that is written is dense.
struct PackedArgs {
    const unsigned short *q, *k, *v;
    long qt, qh, kt, kh, vt, vh;
    int T, Hq, Hk, D;
    float scale;
    // where the tiles are: a table of max_tiles by query and as many by key, or
    // (tiles null) the starts of B sequences
    const int* starts;
    void* tiles;
    int B, max_tiles;
    // the forward pass writes out and, where a backward pass will follow (lse not
    // null), what out's rounding left over, the rows' log-sums and, without
    // tiles, a copy of the starts; the backward pass reads them
    unsigned short *out, *out_lo;
    float* lse;
    int* kept_starts;
    // the backward pass
    const unsigned short* dout;
    long ot, oh;
    float* delta;   // negated
    unsigned short *dq, *dk, *dv;
    // in how many parts the queries may be taken for dk and dv and, where that is
    // more than one, the parts' sums and how many are there for each workgroup's keys
    int parts, counters;
    float* sums;
    int* counts;
};

// The kernel for dk and dv: keys a workgroup, and workgroups that run at once.
constexpr int packed_keys(int D) { return D == 128 ? 128 : 64; }
constexpr int packed_slots(int D) { return D == 128 ? 256 : 3 * 256; }
