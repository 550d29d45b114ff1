// q4_plan.h -- how a launch of linear_q4.cu is divided: shares of the weight
// rows, ranges of k, the ring of stages and the workspace.  Plain host code, so
// that the division and the barriers that rest on it can be checked without a GPU.
#pragma once
#include <cstddef>
#include <cstdint>

namespace rk {

constexpr int Q4_KB = 128;      // columns of a block of K: a row of the 128-byte swizzle
constexpr int Q4_ROWS = 32;     // most activation rows of a pass over the weights
constexpr int Q4_M = 128;       // the MMA's weight rows
constexpr int Q4_STAGES = 8;    // most stages
constexpr int Q4_CODES = 8;     // warps that turn codes into operands
constexpr int Q4_SUMS = 8;      // warps that add up accumulators, in two sets
constexpr int Q4_A_BYTES = Q4_M * Q4_KB;
constexpr int Q4_THREADS = 32 * (2 + Q4_CODES + Q4_SUMS);  // and x copies, products
constexpr int Q4_SMEM = 220 * 1024;

// What the parts of a row stand for.
struct Q4Row {
    float inv;  // 2^9 / the power of two that x was scaled by, as two factors
    float inv2;
    int odd;    // does not fit the parts
    int pad;
};

// How a launch is divided, the same for all of its blocks.
struct Q4Plan {
    int h, pad;          // ranges of k below one another, weight rows set aside for each (128 / h)
    int share;           // most weight rows of a block
    int steps;           // blocks of K of a range
    int sub;             // groups of a block of K: 4, 2, 1
    int mq;              // activation rows of a pass, in fours
    int nc;              // N columns of a range: parts x mq, in eights
    int mma_n;           // N of an MMA
    uint32_t x_bytes;    // of a step: the operand rows [h * nc][128]
    int stages;
    uint32_t s_off, stage;      // shared memory: [128][sub] scales of a stage, a stage
    uint32_t acc_cols, tmem_cols, idesc;
    int accs;                   // accumulators: 4 where they fit, 2
    size_t pass_bytes;   // workspace of a pass
    int pass0;           // first pass of a launch
    long long grid;      // blocks of a pass
    int smem;            // dynamic shared memory of a block
};

inline int q4_parts(size_t type_bytes) { return type_bytes == 4 ? 6 : 3; }
inline int q4_sub(int group) { return group == 32 ? 4 : group == 64 ? 2 : 1; }

// The widths that a pass has whatever the division: activation rows in fours, N columns of a range in eights.
inline void q4_widths(int rows, size_t type_bytes, int& mq, int& nc) {
    const int m = rows < Q4_ROWS ? rows : Q4_ROWS;
    mq = (m + 3) / 4 * 4;
    nc = (q4_parts(type_bytes) * mq + 7) / 8 * 8;
}

inline size_t q4_workspace(int rows, int k, size_t type_bytes) {
    const long long passes = ((long long)rows + Q4_ROWS - 1) / Q4_ROWS, blocks = ((long long)k + Q4_KB - 1) / Q4_KB;
    int mq, nc;
    q4_widths(rows, type_bytes, mq, nc);
    // 4 even ranges of k have up to 3 blocks more than k
    const size_t pass = (size_t)(blocks + 3) * nc * 128 + Q4_ROWS * sizeof(Q4Row);
    return (size_t)passes * ((pass + 255) / 256 * 256);
}

// False where the ring would have too few stages.
inline bool q4_plan(int rows, int n, int k, int group, size_t type_bytes, int sms, Q4Plan& p) {
    p = {};
    const int blocks = (int)(((long long)k + Q4_KB - 1) / Q4_KB);
    // an even share of the weight rows for each SM, in as many rounds as 128 rows a block make it
    p.grid = sms;
    while ((n + p.grid - 1) / p.grid > Q4_M) p.grid += sms;
    if (p.grid > n) p.grid = n;
    p.share = (int)((n + p.grid - 1) / p.grid);
    p.h = p.share <= 32 ? 4 : p.share <= 64 ? 2 : 1;
    while (p.h > blocks) p.h /= 2;
    q4_widths(rows, type_bytes, p.mq, p.nc);
    while (p.h > 1 && p.h * p.nc > 128) p.h /= 2;  // wide ones need no filling: their MMAs take as long as their N
    p.pad = Q4_M / p.h;
    p.steps = (blocks + p.h - 1) / p.h;
    p.sub = q4_sub(group);
    p.x_bytes = (uint32_t)(p.h * p.nc * 128);
    p.mma_n = (p.h * p.nc + 15) / 16 * 16;
    p.acc_cols = (uint32_t)(p.mma_n + 31) / 32 * 32;
    p.accs = 4 * p.acc_cols <= 512 ? 4 : 2;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.accs * p.acc_cols) p.tmem_cols *= 2;
    p.pass_bytes = ((size_t)p.steps * p.x_bytes + Q4_ROWS * sizeof(Q4Row) + 255) / 256 * 256;
    // an MMA of N in sixteens may read eight rows past a stage's operand rows, which the scales' place makes up for
    p.s_off = Q4_A_BYTES + p.x_bytes;
    p.stage = (p.s_off + Q4_M * p.sub * (uint32_t)sizeof(float) + 1023) / 1024 * 1024;
    p.stages = (Q4_SMEM - 1024) / (int)p.stage;
    if (p.stages > Q4_STAGES) p.stages = Q4_STAGES;
    // A wait tells a stage's rounds apart by one bit, so no warp may come to a stage's barrier two rounds early.  A warp
    // of codes at step i knows that step i - Q4_CODES / 2 - stages was used up, because it has waited for that; the
    // round before last of its stage is step i - 2 stages.  It must have been used up too: it is no later when there are
    // Q4_CODES / 2 stages or more, and steps are used up in order where both sets of sums look at every step.  Where
    // they take turns (one group a block of K) a set's own steps are in order only, and the two steps are of the same
    // set when the stages are even in number.
    if (p.sub == 1) p.stages &= ~1;
    if (p.stages < Q4_CODES / 2) return false;
    p.smem = p.stages * (int)p.stage;
    const int red = 2 * Q4_ROWS * Q4_M * 4;
    if (p.smem < red) p.smem = red;
    p.smem += 1024;
    return true;
}

}  // namespace rk
