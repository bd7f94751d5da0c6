// kv8_join.cuh -- who joins the parts of a row tile that several CTAs share
// (kv8_attend.cu).  Plain arithmetic: it also compiles for the host, where
// tests/kv8_join_check.cpp plays it through in any order of the CTAs.
//
// A row tile shared by CTAs c0 .. c1 has a part in each of them.  A CTA that has
// its part counts itself in, and the last one to come joins them: up to kJoinAll
// parts at once, more of them in groups of kJoinGroup consecutive CTAs first,
// whose last one counts the group in.
//
// Where work is shared out by tiles, the CTA that leaves one row tile is often
// the one that enters the next, so a counter must not be reached from both.  A
// group of two parts or more counts at its first CTA, which lies before the last
// CTA of its row tile, and so before all CTAs of the next one; a row tile counts
// at its first CTA in the other half of the counters, likewise.  A group of one
// part would count at that CTA; it needs no count, since its part already lies
// where the groups' results do.
#pragma once

#ifdef __CUDACC__
#define QR_JOIN_FN __host__ __device__ __forceinline__
#else
#define QR_JOIN_FN inline
#endif

namespace qr {

// (Groups from 17 parts up: one sequence of 16,384 tokens 19.5 us instead of 18.7,
// 8 of 500 to 100,000 56.5 instead of 54.6.  Groups of 32: one of 131,072 39.0
// instead of 35.6.)
constexpr int kJoinAll = 32;
constexpr int kJoinGroup = 16;
constexpr int kJoinCtas = 512;  // most CTAs; 2 * kJoinCtas counters, zero between calls

// One count: `n` of them are waited for at counters[counter].
struct JoinStep {
    int counter, n;
};

QR_JOIN_FN bool join_grouped(int c0, int c1) { return c1 - c0 + 1 > kJoinAll; }
// First CTA of the group of CTA `me`.
QR_JOIN_FN int join_group(int c0, int me) { return c0 + (me - c0) / kJoinGroup * kJoinGroup; }

// The step that a CTA with a part begins with: 0, its group; 1, the row tile.
QR_JOIN_FN int join_first(int c0, int c1, int me)
{
    return join_grouped(c0, c1) && join_group(c0, me) < c1 ? 0 : 1;
}

QR_JOIN_FN JoinStep join_step(int step, int c0, int c1, int me)
{
    const int n = c1 - c0 + 1;
    if (step == 0) {
        const int g0 = join_group(c0, me), left = c1 - g0 + 1;
        return {g0, left < kJoinGroup ? left : kJoinGroup};
    }
    return {kJoinCtas + c0, join_grouped(c0, c1) ? (n + kJoinGroup - 1) / kJoinGroup : n};
}

} // namespace qr
