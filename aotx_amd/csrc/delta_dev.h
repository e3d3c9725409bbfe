/* Device parts that the kernels of linear layers share (delta.hip, delta_conv.hip). */
#ifndef AOTX_DELTA_DEV_H
#define AOTX_DELTA_DEV_H

#include "aotx_internal.h"

typedef float aotx_f4 __attribute__((ext_vector_type(4)));
typedef unsigned short aotx_u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short aotx_u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short aotx_u16x8 __attribute__((ext_vector_type(8)));

/* The sequences of a call: rows, positions and slots. offset null: sequence i is row i. */
struct aotx_seqs {
    const unsigned int *offset;
    const unsigned int *pos;
    const unsigned int *agent;
    unsigned int seqs;
    unsigned int tokens;
    unsigned int slots;
    unsigned int *faults;
};

/* One sequence as every lane of a wave sees it. */
struct aotx_seq_view {
    unsigned int start, end;    /* its rows */
    unsigned int slot;
    bool fresh;                 /* starts from zeros */
    bool refused;               /* no slot, or a slot that an earlier sequence has */
};

/* Rows of sequence `lane`, for the first `seqs` lanes of a wave (all 64 call this): in bounds,
 * and none before an earlier sequence's last, whatever the offsets hold. */
static __device__ __forceinline__ void aotx_seq_rows(const aotx_seqs &s, unsigned int *start,
                                                     unsigned int *end)
{
    const unsigned int lane = threadIdx.x & 63u;
    unsigned int b = 0u, e = 0u;
    if (s.offset == nullptr) {
        if (lane < s.seqs) {
            b = lane;
            e = lane + 1u;
        }
    } else {
        if (lane < s.seqs) {
            b = s.offset[lane];
            e = s.offset[lane + 1u];
            b = b < s.tokens ? b : s.tokens;
            e = e < s.tokens ? e : s.tokens;
        }
        for (unsigned int off = 1u; off < s.seqs; off <<= 1) {
            const unsigned int o = (unsigned int)__shfl_up((int)b, off, 64);
            if (lane >= off && o > b) b = o;
        }
        if (e < b) e = b;
    }
    *start = b;
    *end = e;
}

/* Sequence i (wave-uniform), read by all 64 lanes of a wave: lane j looks at sequence j, which
 * tells whether an earlier one with rows has the same slot (at most 64 sequences a call). b and
 * e are the lanes' rows from aotx_seq_rows. */
static __device__ __forceinline__ aotx_seq_view aotx_seq_of(const aotx_seqs &s, unsigned int i,
                                                            unsigned int b, unsigned int e)
{
    const unsigned int lane = threadIdx.x & 63u;
    const unsigned int a = lane < s.seqs ? s.agent[lane] : 0xFFFFFFFFu;
    aotx_seq_view v;
    v.start = (unsigned int)__builtin_amdgcn_readlane((int)b, (int)i);
    v.end = (unsigned int)__builtin_amdgcn_readlane((int)e, (int)i);
    v.slot = (unsigned int)__builtin_amdgcn_readlane((int)a, (int)i);
    const unsigned long long same = __ballot(lane < i && b < e && a == v.slot);
    v.refused = v.slot >= s.slots || same != 0ull;
    v.fresh = s.pos[i] == 0u;
    return v;
}

/* Sum over a wave. */
static __device__ __forceinline__ float aotx_wave_sum(float v)
{
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

/* x / (1 + exp(-x)) */
static __device__ __forceinline__ float aotx_silu(float x)
{
    return x / (1.0f + expf(-x));
}

/* g = decay softplus(a + dt), at most 0; below -1000 its exponential is 0 all the same and
 * sums of it stay finite. A NaN stays one. */
static __device__ __forceinline__ float aotx_delta_gate(float a, float dt, float decay)
{
    const float x = a + dt;
    float g = decay * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
    if (x != x) g = x;
    if (g > 0.0f) g = 0.0f;
    if (g < -1000.0f) g = -1000.0f;
    return g;
}

/* The faults counter of the device state, made on first use; null when this stream is being
 * captured and no call has made it yet (the caller then refuses). */
static inline unsigned int *aotx_faults(void *stream)
{
    aotx_state *st = aotx_state_existing();
    if (st == nullptr) {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (stream != nullptr) AOTX_CHECK(hipStreamIsCapturing(aotx_stream(stream), &status));
        if (status != hipStreamCaptureStatusNone) {
            fprintf(stderr, "aotx: the first call of a process cannot be captured\n");
            return nullptr;
        }
        st = aotx_state_device();
    }
    return &st->faults;
}

static inline bool aotx_aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

#endif
