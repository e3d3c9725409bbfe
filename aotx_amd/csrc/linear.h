/* The product of many rows with an epilogue of its own (linear.hip), for aotx_q8_linear (rgemv.hip). */
#ifndef AOTX_LINEAR_H
#define AOTX_LINEAR_H

#include "rgemv.h"

/* What aotx_q8_linear does with a product's sums: y = act(sum + bias) [* (up sum + up_bias)] + resid. */
struct aotx_linear_epi {
    static constexpr bool LINEAR = true;
    const float *bias, *up_bias, *resid;
    unsigned int ldr, act, half;
};

/* Tiles of 256 weight rows (of a pair: 128 of each) by `bm` batch rows. On each of the 8 XCDs
 * `whole` workgroups take a tile each, rounds of 32, and the tiles that are left are split along k where
 * CUs would else have nothing to do. */
struct aotx_lgemm_plan {
    unsigned int bm;            /* 256, 192 or 128 */
    unsigned int ny;            /* row blocks */
    unsigned int groups;        /* of weight rows */
    unsigned int tiles;         /* of one XCD */
    unsigned int whole, splits, qps;
};

/* The plan of m rows; returns the nanoseconds that it should take. */
unsigned long long aotx_lgemm_choose(aotx_lgemm_plan *p, unsigned int n, unsigned int k, unsigned int m, bool gated, bool file);
size_t aotx_lgemm_partial_bytes(const aotx_lgemm_plan &p);
void aotx_lgemm_launch(const aotx_lgemm_plan &p, const aotx_rgemv_args &a, const aotx_linear_epi &e, hipStream_t s);

#endif
