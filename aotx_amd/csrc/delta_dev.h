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

/* The call's sequences as a wave holds them, sequence j in lane j (at most 64 a call). */
struct aotx_seq_lanes {
    unsigned int start, end;    /* rows: in bounds, none before an earlier sequence's last, whatever the offsets hold */
    unsigned int slot, pos;
};

static __device__ __forceinline__ aotx_seq_lanes aotx_seqs_read(const aotx_seqs &s)
{
    const unsigned int lane = threadIdx.x & 63u;
    aotx_seq_lanes v = {0u, 0u, 0xFFFFFFFFu, 0u};
    if (lane < s.seqs) {
        v.start = s.offset != nullptr ? s.offset[lane] : lane;
        v.end = s.offset != nullptr ? s.offset[lane + 1u] : lane + 1u;
        v.slot = s.agent[lane];
        v.pos = s.pos[lane];
    }
    if (s.offset != nullptr) {
        v.start = v.start < s.tokens ? v.start : s.tokens;
        v.end = v.end < s.tokens ? v.end : s.tokens;
        if (lane >= s.seqs) v.start = v.end = 0u;
        for (unsigned int off = 1u; off < s.seqs; off <<= 1) {
            const unsigned int o = (unsigned int)__shfl_up((int)v.start, off, 64);
            if (lane >= off && o > v.start) v.start = o;
        }
        if (v.end < v.start) v.end = v.start;
    }
    return v;
}

/* Sequence i (wave-uniform): a ballot tells whether an earlier one with rows has the same slot. */
static __device__ __forceinline__ aotx_seq_view aotx_seq_of(const aotx_seqs &s, unsigned int i, const aotx_seq_lanes &l)
{
    const unsigned int lane = threadIdx.x & 63u;
    aotx_seq_view v;
    v.start = (unsigned int)__builtin_amdgcn_readlane((int)l.start, (int)i);
    v.end = (unsigned int)__builtin_amdgcn_readlane((int)l.end, (int)i);
    v.slot = (unsigned int)__builtin_amdgcn_readlane((int)l.slot, (int)i);
    const unsigned long long same = __ballot(lane < i && l.start < l.end && l.slot == v.slot);
    v.refused = v.slot >= s.slots || same != 0ull;
    v.fresh = (unsigned int)__builtin_amdgcn_readlane((int)l.pos, (int)i) == 0u;
    return v;
}

/* Sum over a wave. */
static __device__ __forceinline__ float aotx_wave_sum(float v)
{
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

/* Running sum of 64 lanes' values, in 64 bits. */
template <int CTRL, int ROWS>
static __device__ __forceinline__ double aotx_dpp_add(double v)
{
    const long long b = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, false);
    return v + __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned int)lo);
}
static __device__ __forceinline__ double aotx_wave_scan(double v)
{
    v = aotx_dpp_add<0x111, 0xF>(v);        /* lanes 1, 2, 4 and 8 before, within rows of 16 */
    v = aotx_dpp_add<0x112, 0xF>(v);
    v = aotx_dpp_add<0x114, 0xF>(v);
    v = aotx_dpp_add<0x118, 0xF>(v);
    v = aotx_dpp_add<0x142, 0xA>(v);        /* the last lane of row 0 to row 1, of row 2 to row 3 */
    v = aotx_dpp_add<0x143, 0xC>(v);        /* lane 31 to rows 2 and 3 */
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
