// seq_step.hip -- attention that decays with distance, one token of many rows (include/pvder_sequence.h: pvder_seq_step_run).
//
//   S = g S + k v^T,   o = scale S^T q        per row n and head h, S [dk][dv] fp32 in memory
//
// Bound: the state, read and written once: 8 dk dv bytes of 8 dk dv + (2 dk + 2 dv) elements.  A lane holds 16 bytes of a row of
// S and walks down the rows; the lanes beside it hold the rest of the row, so that a wave reads whole rows.
// Measured: 65 536 envs x 4 heads of 32 x 32, fp32, 404 us, 2.28 GB at 5.65 TB/s; 1001 envs x 3 heads of 48 x 80, bf16, 17 us, 93 MB at
// 5.4 TB/s; one env 3.7 us, which is what a launch takes.
#include "seq_common.hpp"

namespace {

using namespace pvder_seq;

constexpr int kBlock = 256;

// W columns per lane, CL lanes to a row of columns, WAVES waves to a cell (n, h)
template <typename T, int W, int CL, int WAVES> __global__ __launch_bounds__(kBlock) void seq_step_kernel(const pvder_seq_step a) {
    constexpr int RL = 64 / CL * WAVES;                    // rows of S that are in hand side by side
    __shared__ float part[WAVES > 1 ? WAVES : 1][CL * W];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long cell = WAVES > 1 ? (long long)blockIdx.x : blockIdx.x * (long long)(kBlock / 64) + wave;
    const bool on = cell < (long long)a.N * a.H;
    if (WAVES == 1 && !on) return;
    const long long n = cell / a.H;
    const int h = (int)(cell - n * a.H);
    const int cl = lane % CL, rl = (WAVES > 1 ? wave * (64 / CL) : 0) + lane / CL;
    const T *q = (const T *)a.q + n * a.q_n + h * a.q_h;
    const T *k = (const T *)a.k + n * a.k_n + h * a.k_h;
    const T *v = (const T *)a.v + n * a.v_n + h * a.v_h;
    T *o = (T *)a.o + n * a.o_n + h * a.o_h;
    float *S = a.state + cell * ((long long)a.dk * a.dv);
    const uint8_t start = a.starts ? a.starts[n * a.starts_n] : 0;
    const float g = power(log2_decay(a.log_decay[h]), 1);
    const bool fresh = (start != 0) | (g == 0.f);          // (a weight of zero clears what is not finite, too)
    for (int c0 = 0; c0 < a.dv; c0 += CL * W) {
        const int c = c0 + cl * W;
        const bool in = c < a.dv;                          // (W = 4 only where dv is a multiple of 4)
        float vv[W], acc[W];
#pragma unroll
        for (int e = 0; e < W; ++e) { vv[e] = in ? (float)v[c + e] : 0.f; acc[e] = 0.f; }
        if (in) {
#pragma unroll 4
            for (int d = rl; d < a.dk; d += RL) {
                float s[W];
                float *p = S + (long long)d * a.dv + c;
                if constexpr (W == 4) { const f4 t = *(const f4 *)p; s[0] = t.x; s[1] = t.y; s[2] = t.z; s[3] = t.w; }
                else s[0] = *p;
                const float kd = (float)k[d], qd = (float)q[d];
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    s[e] = __builtin_fmaf(kd, vv[e], fresh ? 0.f : g * s[e]);
                    acc[e] = __builtin_fmaf(qd, s[e], acc[e]);
                }
                if constexpr (W == 4) *(f4 *)p = f4{s[0], s[1], s[2], s[3]};
                else *p = s[0];
            }
        }
#pragma unroll
        for (int e = 0; e < W; ++e)
#pragma unroll
            for (int x = CL; x < 64; x <<= 1) acc[e] += __shfl_xor(acc[e], x, 64);
        if constexpr (WAVES > 1) {
            if (lane < CL)
#pragma unroll
                for (int e = 0; e < W; ++e) part[wave][cl * W + e] = acc[e];
            __syncthreads();
            if (wave == 0 && lane < CL && in)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    float t = part[0][cl * W + e];
#pragma unroll
                    for (int w = 1; w < WAVES; ++w) t += part[w][cl * W + e];
                    o[c + e] = (T)(t * a.scale);
                }
            __syncthreads();
        } else if (lane < CL && in) {
#pragma unroll
            for (int e = 0; e < W; ++e) o[c + e] = (T)(acc[e] * a.scale);
        }
    }
}

// a large cell is shared by the four waves of a block: one wave would read it in dk / 2 dependent rounds
bool shared(const pvder_seq_step &a) { return (long long)a.dk * a.dv > 4096; }

template <typename T, int W, int CL> int launch(const pvder_seq_step &a, hipStream_t st) {
    const long long cells = (long long)a.N * a.H, blocks = shared(a) ? cells : (cells + kBlock / 64 - 1) / (kBlock / 64);
    if (shared(a)) seq_step_kernel<T, W, CL, kBlock / 64><<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(a);
    else seq_step_kernel<T, W, CL, 1><<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -(int)e;
}

template <typename T> int pick(const pvder_seq_step &a, hipStream_t st) {
    if (a.dv % 4 == 0 && ((uintptr_t)a.state & 15) == 0) {
        if (a.dv <= 16) return launch<T, 4, 4>(a, st);
        if (a.dv <= 32) return launch<T, 4, 8>(a, st);
        if (a.dv <= 64) return launch<T, 4, 16>(a, st);
        return launch<T, 4, 32>(a, st);
    }
    if (a.dv <= 16) return launch<T, 1, 16>(a, st);
    if (a.dv <= 32) return launch<T, 1, 32>(a, st);
    return launch<T, 1, 64>(a, st);
}

}  // namespace

extern "C" int pvder_seq_step_run(const pvder_seq_step *a, void *stream) {
    if (!a || a->N < 0 || a->H < 1 || a->dk < 1 || a->dv < 1 || a->dk > PVDER_SEQ_MAX_HEAD || a->dv > PVDER_SEQ_MAX_HEAD) return kEinval;
    if (a->dtype != PVDER_SEQ_F32 && a->dtype != PVDER_SEQ_BF16) return kEinval;
    if (a->N == 0) return 0;
    if (!a->q || !a->k || !a->v || !a->o || !a->state || !a->log_decay) return kEinval;
    // as many rows to a launch as its threads can be counted for
    const long long most = kMostThreads / kBlock * (shared(*a) ? 1 : kBlock / 64) / a->H;
    if (most < 1) return kEinval;
    const long long es = a->dtype == PVDER_SEQ_BF16 ? 2 : 4;
    for (long long n = 0; n < a->N; n += most) {
        pvder_seq_step part = *a;
        part.N = (int32_t)(a->N - n < most ? a->N - n : most);
        part.q = (const char *)a->q + n * a->q_n * es;
        part.k = (const char *)a->k + n * a->k_n * es;
        part.v = (const char *)a->v + n * a->v_n * es;
        part.o = (char *)a->o + n * a->o_n * es;
        part.state = a->state + n * a->H * ((long long)a->dk * a->dv);
        if (a->starts) part.starts = a->starts + n * a->starts_n;
        const int rc = a->dtype == PVDER_SEQ_BF16 ? pick<__bf16>(part, (hipStream_t)stream) : pick<float>(part, (hipStream_t)stream);
        if (rc) return rc;
    }
    return 0;
}
