/* The rotary turn that aotx_rope_axes (hybrid_rows.hip) and aotx_kv_append (append.hip) make: the
 * pairs' frequencies and axes, made on the host, and a lane's eight values of a head. */
#ifndef AOTX_ROPE_DEV_H
#define AOTX_ROPE_DEV_H

#include "delta_dev.h"
#include "../../include/aotx_hybrid.h"

#include <math.h>

struct aotx_rope_turns {
    double turns[64];           /* of pair i at place 1: theta^(-2i/r) / (2 pi) */
    unsigned char axis[64];
};

/* Whether a head of head_dim values can turn so. */
static inline bool aotx_rope_ok(const aotx_rope_how *how, unsigned int head_dim)
{
    const unsigned int r = how->rope_dim;
    if (r == 0u || r % 8u != 0u || r > head_dim) return false;
    if (how->pairs != AOTX_ROPE_PAIRS_SPLIT && how->pairs != AOTX_ROPE_PAIRS_ADJACENT) return false;
    if (how->axes == 0u || how->axes > AOTX_ROPE_AXES_MAX) return false;
    if (how->order != AOTX_ROPE_AXES_RUNS && how->order != AOTX_ROPE_AXES_TURN) return false;
    if (!(how->theta > 0.0f) || !isfinite(how->theta) || !(how->eps >= 0.0f)) return false;
    unsigned long long sum = 0u;
    for (unsigned int i = 0; i < how->axes; ++i) sum += how->span[i];
    return sum == r / 2u;
}

static inline void aotx_rope_fill(const aotx_rope_how *how, aotx_rope_turns *p)
{
    const unsigned int r = how->rope_dim;
    /* powers of one step: 64 products round by less than 2^-46 of a frequency */
    const double step = pow((double)how->theta, -2.0 / (double)r);
    double turn = 0.15915494309189533577;       /* 1 / (2 pi) */
    unsigned int axis = 0u, left = how->span[0];
    for (unsigned int i = 0; i < 64u; ++i, turn *= step) {
        p->turns[i] = turn;
        p->axis[i] = 0u;
        if (i >= r / 2u) continue;
        if (how->order == AOTX_ROPE_AXES_TURN) {
            const unsigned int a = i % how->axes;
            p->axis[i] = (unsigned char)(i < how->axes * how->span[a] ? a : 0u);
        } else {
            while (left == 0u) left = how->span[++axis];
            --left;
            p->axis[i] = (unsigned char)axis;
        }
    }
}

/* The fraction of a turn that a pair makes at `place` (64 bits hold what far places need). */
static __device__ __forceinline__ float aotx_rope_angle(double place, double turns, const float *factor, unsigned int i)
{
    double a = place * turns;
    if (factor != nullptr) a /= (double)factor[i];
    return (float)(a - floor(a));               /* [0, 1] turns */
}

/* A lane's eight values, x0 at lo.. and x1 at hi.., turned by the cosines c and sines s of its four
 * pairs and rounded. */
static __device__ __forceinline__ void aotx_rope_pairs(unsigned int pairs, const aotx_f4 &x0, const aotx_f4 &x1,
                                                       const float *c, const float *s, aotx_u16x4 &y0, aotx_u16x4 &y1)
{
    if (pairs == AOTX_ROPE_PAIRS_SPLIT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y0[e] = aotx_f2h(x0[e] * c[e] - x1[e] * s[e]);
            y1[e] = aotx_f2h(x0[e] * s[e] + x1[e] * c[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            y0[2 * e] = aotx_f2h(x0[2 * e] * c[e] - x0[2 * e + 1] * s[e]);
            y0[2 * e + 1] = aotx_f2h(x0[2 * e] * s[e] + x0[2 * e + 1] * c[e]);
            y1[2 * e] = aotx_f2h(x1[2 * e] * c[2 + e] - x1[2 * e + 1] * s[2 + e]);
            y1[2 * e + 1] = aotx_f2h(x1[2 * e] * s[2 + e] + x1[2 * e + 1] * c[2 + e]);
        }
    }
}

#endif
