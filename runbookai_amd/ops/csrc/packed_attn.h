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
    // the tiles: a table of max_tiles by query, as many by key, and how many pairs
    // of them meet.  It is built from the starts of B sequences or (search) found
    // by the forward kernel, which leaves it where a backward pass will follow.
    const int* starts;
    void* tiles;
    int B, max_tiles, search;
    // the forward pass writes out and, where a backward pass will follow (lse not
    // null), what out's rounding left over and the rows' log-sums
    unsigned short *out, *out_lo;
    float* lse;
    // the backward pass
    const unsigned short* dout;
    long ot, oh;
    float* delta;   // negated
    unsigned short *dq, *dk, *dv;
    // in how many parts the queries may be taken for dk and dv and, where that is
    // more than one, the parts' sums (dk and dv in fp32, each) and how many are there
    // for each workgroup's keys
    int parts, counters;
    float* sums;
    int* counts;
};

// The kernel for dk and dv: keys a workgroup (and queries a step), workgroups that
// run at once, and steps that a workgroup must have over its share to be split.
constexpr int packed_keys(int D) { return D == 128 ? 128 : 64; }
constexpr int packed_slots(int D) { return D == 128 ? 256 : 3 * 256; }
constexpr int packed_worth(int D) { return D == 128 ? 8 : 16; }
