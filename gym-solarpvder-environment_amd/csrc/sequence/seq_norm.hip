// seq_norm.hip -- the residual stream between two blocks (include/pvder_sequence.h: pvder_seq_norm_forward / _backward).
//
//   forward    n = y ry post,  u = sigmoid(gate) n,  h' = h + scale u,  x = h' rh pre          ry, rh: one over the rows' rms
//   backward   d = dh + rh (dx pre - h' rh^2 mean(dx pre h'))          the gradient of h, and of h' from both sides
//              dn = d scale sigmoid post,   dy = ry (dn - y ry^2 mean(dn y)),   dgate = d scale n sigmoid (1 - sigmoid)
//              dpost = sum d scale sigmoid y ry,   dpre = sum dx h' rh,   dscale = sum d u     over the rows
//
// Bound: bytes; 3 tensors in and 2 out forward, 5 in and 3 out backward.  TPR lanes hold a row in registers, so each tensor is
// read once; the backward pass takes h' from h, y and gate again (read anyway) and not from its rounded copy.  The sums over the
// rows are kept in registers by column, joined per block in LDS, and over the blocks by a second kernel in a fixed order.
// Measured: forward, 65 536 x 128, fp32, 27 us (its 168 MB are in the last-level cache), 16 384 x 2048, bf16, 66 us, 5.1 TB/s, 16 384 x
// 8192, 271 us, 5.0 TB/s; backward with the sums, 262 144 x 64, fp32, 113 us, 4.8 TB/s, 16 384 x 2048, bf16, 145 us, 3.7 TB/s (50 vector
// instructions an element between two sums over the row), 16 384 x 8192, bf16, 781 us, 2.7 TB/s (one block on a CU, so nothing runs
// while it waits for a row).  Rows fetched one ahead were slower everywhere: the registers that they take cost a third of the waves.
#include "seq_common.hpp"

namespace {

using namespace pvder_seq;

// threads of a block: 256 where a wave holds whole rows, else one row's
constexpr int block_of(int tpr) { return tpr > 64 ? tpr : 256; }

template <typename T, int NV> struct Row {
    static constexpr int V = Vec<T>::N, E = V * NV;
    float e[E];
};

// lane t of TPR holds the vectors t, t + TPR, ...;  EVEN: the width is a multiple of a vector, which then is there whole or not at all
template <typename T, bool EVEN> __device__ __forceinline__ typename Vec<T>::type load_vec(const T *row, int d, int D) {
    if constexpr (EVEN) {
        u4 u;
        __builtin_memcpy(&u, row + (d < D ? d : 0), 16);
        return __builtin_bit_cast(typename Vec<T>::type, d < D ? u : u4{0u, 0u, 0u, 0u});
    } else {
        return load_row<T>(row, d, D);
    }
}
template <typename T, bool EVEN> __device__ __forceinline__ void store_vec(T *row, int d, int D, typename Vec<T>::type f) {
    if constexpr (EVEN) {
        if (d < D) __builtin_memcpy(row + d, &f, 16);
    } else {
        store_row<T>(row, d, D, f);
    }
}
template <bool EVEN, typename T, int TPR, int NV> __device__ __forceinline__ void load(Row<T, NV> &r, const T *row, int t, int D) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const typename Vec<T>::type f = load_vec<T, EVEN>(row, (i * TPR + t) * V, D);
#pragma unroll
        for (int e = 0; e < V; ++e) r.e[i * V + e] = (float)f[e];
    }
}
template <bool EVEN, typename T, int TPR, int NV> __device__ __forceinline__ void store(T *row, const Row<T, NV> &r, int t, int D) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        typename Vec<T>::type f;
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (T)r.e[i * V + e];
        store_vec<T, EVEN>(row, (i * TPR + t) * V, D, f);
    }
}
// a row of fp32 weights: zeros behind the width, `otherwise` where there is none
template <bool EVEN, typename T, int TPR, int NV> __device__ __forceinline__ void load_param(Row<T, NV> &r, const float *p, int t, int D, float otherwise) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const int d = (i * TPR + t) * V + k;
            f4 f;
            if (p) f = load_vec<float, EVEN>(p, d, D);
            else f = d < D ? f4{otherwise, otherwise, otherwise, otherwise} : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) r.e[i * V + k + e] = f[e];
        }
}

// what stands before is finished before what stands behind begins: keeps the weights of one vector in registers at a time
__device__ __forceinline__ void apart() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// sum over the TPR lanes of a row; TPR > 64: over the whole block (every lane of it calls)
template <int TPR> __device__ __forceinline__ float row_sum(float x, float *lds) {
#pragma unroll
    for (int k = 1; k < (TPR < 64 ? TPR : 64); k <<= 1) x += __shfl_xor(x, k, 64);
    if constexpr (TPR > 64) {
        __syncthreads();                                   // (the words of the sum before have been read)
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = lds[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) x += lds[w];
    }
    return x;
}

// sigmoid(z) and sigmoid(z) (1 - sigmoid(z)), without cancellation.  t is below 1, and zero where it would be no normal number.
__device__ __forceinline__ void sigmoids(float z, float &s, float &sc) {
    const float t = __builtin_amdgcn_exp2f(-fabsf(z) * 1.44269504088896340736f), r = __builtin_amdgcn_rcpf(1.f + t);
    s = z >= 0.f ? r : t * r;
    sc = t * r * r;
}

// Rows go round the blocks and the weights stay in registers: at a width of 2048 they are as many bytes as a row of all tensors.
template <typename T, int TPR, int NV, bool EVEN> __global__ __launch_bounds__(block_of(TPR)) void seq_norm_forward_kernel(const pvder_seq_norm a) {
    constexpr int BLOCK = block_of(TPR), RPB = BLOCK / TPR, E = Row<T, NV>::E;
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    const int t = threadIdx.x % TPR, D = a.width, grp = threadIdx.x / TPR;
    const float inv = 1.f / (float)D;
    Row<T, NV> post, pre, scale;
    load_param<EVEN, T, TPR, NV>(post, a.post, t, D, 1.f);
    load_param<EVEN, T, TPR, NV>(scale, a.scale, t, D, 1.f);
    load_param<EVEN, T, TPR, NV>(pre, a.pre, t, D, 1.f);
    // (every lane of a block takes as many turns: sums over more than a wave have a barrier in them)
    for (long long r0 = blockIdx.x * (long long)RPB; r0 < a.rows; r0 += gridDim.x * (long long)RPB) {
        const bool on = r0 + grp < a.rows;
        const long long r = on ? r0 + grp : r0;
        Row<T, NV> y, h, z;
        load<EVEN, T, TPR, NV>(y, (const T *)a.y + r * a.y_r, t, D);
        load<EVEN, T, TPR, NV>(h, (const T *)a.h + r * a.h_r, t, D);
        if (a.gate) load<EVEN, T, TPR, NV>(z, (const T *)a.gate + r * a.gate_r, t, D);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = __builtin_fmaf(y.e[e], y.e[e], s);
        const float ry = rsqrtf(row_sum<TPR>(s, lds) * inv + a.eps);
        s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float u = y.e[e] * ry * post.e[e];
            if (a.gate) { float sg, sc; sigmoids(z.e[e], sg, sc); u *= sg; }
            h.e[e] = __builtin_fmaf(scale.e[e], u, h.e[e]);
            s = __builtin_fmaf(h.e[e], h.e[e], s);
        }
        const float rh = rsqrtf(row_sum<TPR>(s, lds) * inv + a.eps);
        if (!on) continue;                                 // (the block's last turn)
        store<EVEN, T, TPR, NV>((T *)a.h_out + r * D, h, t, D);
#pragma unroll
        for (int e = 0; e < E; ++e) h.e[e] *= rh * pre.e[e];
        store<EVEN, T, TPR, NV>((T *)a.x_out + r * D, h, t, D);
        if (a.stats && t == 0) { a.stats[2 * r] = ry; a.stats[2 * r + 1] = rh; }
    }
}

template <typename T, int TPR, int NV, bool EVEN> __global__ __launch_bounds__(block_of(TPR)) __attribute__((amdgpu_waves_per_eu(TPR == 512 && Row<T, NV>::E == 8 ? 4 : 1)))
void seq_norm_backward_kernel(const pvder_seq_norm a) {
    constexpr int BLOCK = block_of(TPR), RPB = BLOCK / TPR, V = Vec<T>::N, E = Row<T, NV>::E;
    typedef typename Vec<T>::type vec;
    // TWICE, rows of over 2048: h' and the sigmoid are taken a second time instead of held, so that two blocks of eight waves find room on a
    // CU: 16384 x 4096, bf16, 442 us -> 303.  LEAN, over 4096 (16 elements a lane): the weights come from L2 a vector at a time, too.
    constexpr bool LEAN = E > 8, TWICE = TPR == 512;
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    __shared__ float sums[RPB > 1 ? RPB * TPR * E : 1];
    const int t = threadIdx.x % TPR, D = a.width, grp = threadIdx.x / TPR;
    Row<T, NV> gpost, gpre, gscale;
    Row<T, LEAN ? 1 : NV> post, pre, scale;                // (LEAN: those of one vector at a time)
    auto weights = [&](int i) {
        load_param<EVEN, T, TPR, LEAN ? 1 : NV>(post, a.post, i * TPR + t, D, 1.f);
        load_param<EVEN, T, TPR, LEAN ? 1 : NV>(pre, a.pre, i * TPR + t, D, 1.f);
        load_param<EVEN, T, TPR, LEAN ? 1 : NV>(scale, a.scale, i * TPR + t, D, 1.f);
    };
    if constexpr (!LEAN) weights(0);
#pragma unroll
    for (int e = 0; e < E; ++e) gpost.e[e] = gpre.e[e] = gscale.e[e] = 0.f;
    const float inv = 1.f / (float)D;
    for (long long r0 = blockIdx.x * (long long)RPB; r0 < a.rows; r0 += gridDim.x * (long long)RPB) {
        const bool on = r0 + grp < a.rows;
        const long long r = on ? r0 + grp : r0;
        vec y[NV], h[NV], z[NV], dh[NV], dx[NV];
        auto row = [&](vec *f, const void *p, int64_t stride) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (p) f[i] = load_vec<T, EVEN>((const T *)p + r * stride, (i * TPR + t) * V, D);
                else f[i] = __builtin_bit_cast(vec, u4{0u, 0u, 0u, 0u});
            }
        };
        row(y, a.y, a.y_r);
        row(h, a.h, a.h_r);
        row(z, a.gate, a.gate_r);
        row(dx, a.dx, a.dx_r);
        row(dh, a.dh, a.dh_r);
        const float ry = a.stats[2 * r], rh = a.stats[2 * r + 1];
        Row<T, TWICE ? 1 : NV> hn, sg, sc;
        Row<T, NV> dn;
        auto branch = [&](int i, int k) {                   // element k of vector i of h', the sigmoid and its derivative
            const int e = TWICE ? k : i * V + k, p = LEAN ? k : i * V + k;
            sg.e[e] = 1.f;
            sc.e[e] = 0.f;
            if (a.gate) sigmoids((float)z[i][k], sg.e[e], sc.e[e]);
            hn.e[e] = __builtin_fmaf(scale.e[p], (float)y[i][k] * ry * post.e[p] * sg.e[e], (float)h[i][k]);
        };
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (LEAN) weights(i);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int e = TWICE ? k : i * V + k, p = LEAN ? k : i * V + k;
                branch(i, k);
                s = __builtin_fmaf((float)dx[i][k] * pre.e[p], hn.e[e], s);
            }
            if constexpr (LEAN) apart();
        }
        const float A = row_sum<TPR>(s, lds) * inv * rh * rh;
        if constexpr (TWICE) {                             // (so that the compiler does not hold them after all)
#pragma unroll
            for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(z[i]), "+v"(y[i]), "+v"(h[i]));
        }
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (LEAN) weights(i);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int e = TWICE ? k : i * V + k, p = LEAN ? k : i * V + k, x0 = i * V + k;
                if constexpr (TWICE) branch(i, k);
                const float x = (float)dx[i][k], n0 = (float)y[i][k] * ry, n = n0 * post.e[p];
                const float d = __builtin_fmaf(rh, x * pre.e[p] - hn.e[e] * A, (float)dh[i][k]), du = d * scale.e[p];
                if (on) {                                  // (a row past the end stands in for the block's first)
                    gpre.e[x0] = __builtin_fmaf(x * hn.e[e], rh, gpre.e[x0]);
                    gscale.e[x0] = __builtin_fmaf(d, n * sg.e[e], gscale.e[x0]);
                    gpost.e[x0] = __builtin_fmaf(du * sg.e[e], n0, gpost.e[x0]);
                }
                z[i][k] = (T)(sc.e[e] * du * n);
                dh[i][k] = (T)d;
                dn.e[x0] = du * sg.e[e] * post.e[p];
                s = __builtin_fmaf(dn.e[x0], (float)y[i][k], s);
            }
            if constexpr (LEAN) apart();
        }
        const float B = row_sum<TPR>(s, lds) * inv * ry * ry;
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int d0 = (i * TPR + t) * V;
            vec f;
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = (T)(ry * (dn.e[i * V + k] - (float)y[i][k] * B));
            store_vec<T, EVEN>((T *)a.dh_out + r * D, d0, D, dh[i]);
            store_vec<T, EVEN>((T *)a.dy_out + r * D, d0, D, f);
            if (a.gate) store_vec<T, EVEN>((T *)a.dgate_out + r * D, d0, D, z[i]);
        }
    }
    if (!a.dparam) return;
    float *out = (gridDim.x > 1 ? a.workspace : a.dparam) + blockIdx.x * 3ll * D;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        Row<T, NV> &v = k == 0 ? gpost : (k == 1 ? gpre : gscale);
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) sums[grp * (TPR * E) + (i * TPR + t) * V + e] = v.e[i * V + e];
            __syncthreads();
            for (int d = threadIdx.x; d < D; d += BLOCK) {
                float x = sums[d];
                for (int g = 1; g < RPB; ++g) x += sums[g * (TPR * E) + d];
                out[k * D + d] = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int d = (i * TPR + t) * V + e;
                    if (d < D) out[k * D + d] = v.e[i * V + e];
                }
        }
    }
}

// sums over the blocks' partial rows, 32 columns and 8 parts of the rows to a block
__global__ __launch_bounds__(256) void seq_norm_sum_kernel(const float *__restrict__ part, float *__restrict__ out, int n, int cols) {
    __shared__ float lds[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    float s = 0.f;
    if (col < cols)
#pragma unroll 8
        for (int r = g; r < n; r += 8) s += part[(long long)r * cols + col];
    lds[g][c] = s;
    __syncthreads();
    if (g == 0 && col < cols) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += lds[k][c];
        out[col] = s;
    }
}

// lanes to a row: the fewest that hold it at 8 elements a lane, 4 at least; 512 lanes hold 16 where they have to
int lanes_of(int width) {
    int tpr = 4;
    while (tpr * 8 < width && tpr < 512) tpr <<= 1;
    return tpr;
}
int rows_per_block(int tpr) { return block_of(tpr) / tpr; }
// blocks for `rows` rows, `waves` of them on each of the 256 CUs at most, all with as many turns
long long blocks_of(long long rows, int tpr, int waves) {
    const long long need = (rows + rows_per_block(tpr) - 1) / rows_per_block(tpr), most = 256ll * waves * 64 / block_of(tpr);
    const long long turns = (need + most - 1) / most;
    return (need + turns - 1) / turns;
}
// Waves on a CU: a whole number of blocks that it holds at once.  (Backward, 512 lanes to a row: 12 waves are one and a half blocks,
// 16384 x 5000, fp32, 1172 us, 16 waves 946.)
constexpr int kForwardWaves = 24;
constexpr int backward_waves(int tpr) { return tpr == 512 ? 16 : 12; }

template <typename T, int TPR, int NV, bool EVEN> void start(const pvder_seq_norm &a, bool back, hipStream_t st) {
    constexpr int BLOCK = block_of(TPR);
    const unsigned blocks = (unsigned)blocks_of(a.rows, TPR, back ? backward_waves(TPR) : kForwardWaves);
    if (back) {
        seq_norm_backward_kernel<T, TPR, NV, EVEN><<<dim3(blocks), dim3(BLOCK), 0, st>>>(a);
        if (a.dparam && blocks > 1)
            seq_norm_sum_kernel<<<dim3((3 * a.width + 31) / 32), dim3(256), 0, st>>>(a.workspace, a.dparam, (int)blocks, 3 * a.width);
    } else {
        seq_norm_forward_kernel<T, TPR, NV, EVEN><<<dim3(blocks), dim3(BLOCK), 0, st>>>(a);
    }
}

template <typename T, int TPR, int PER_LANE = 8> int run(const pvder_seq_norm &a, bool back, hipStream_t st) {
    constexpr int NV = PER_LANE / Vec<T>::N;
    if (a.width % Vec<T>::N == 0) start<T, TPR, NV, true>(a, back, st);
    else start<T, TPR, NV, false>(a, back, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -(int)e;
}

template <typename T> int pick(const pvder_seq_norm &a, bool back, hipStream_t st) {
    switch (lanes_of(a.width)) {
        case 4: return run<T, 4>(a, back, st);
        case 8: return run<T, 8>(a, back, st);
        case 16: return run<T, 16>(a, back, st);
        case 32: return run<T, 32>(a, back, st);
        case 64: return run<T, 64>(a, back, st);
        case 128: return run<T, 128>(a, back, st);
        case 256: return run<T, 256>(a, back, st);
        default: return a.width <= 4096 ? run<T, 512>(a, back, st) : run<T, 512, 16>(a, back, st);
    }
}

bool ok(const pvder_seq_norm *a) {
    return a && a->rows >= 0 && a->width >= 1 && a->width <= PVDER_SEQ_MAX_WIDTH && a->eps >= 0.f &&
           (a->dtype == PVDER_SEQ_F32 || a->dtype == PVDER_SEQ_BF16);
}

}  // namespace

extern "C" int64_t pvder_seq_norm_workspace(const pvder_seq_norm *a) {
    if (!ok(a)) return kEinval;
    if (!a->dparam || a->rows == 0) return 0;
    const long long blocks = blocks_of(a->rows, lanes_of(a->width), backward_waves(lanes_of(a->width)));
    return blocks > 1 ? blocks * 3 * a->width : 0;
}

extern "C" int pvder_seq_norm_forward(const pvder_seq_norm *a, void *stream) {
    if (!ok(a)) return kEinval;
    if (a->rows == 0) return 0;
    if (!a->h || !a->y || !a->post || !a->pre || !a->h_out || !a->x_out) return kEinval;
    return a->dtype == PVDER_SEQ_BF16 ? pick<__bf16>(*a, false, (hipStream_t)stream) : pick<float>(*a, false, (hipStream_t)stream);
}

extern "C" int pvder_seq_norm_backward(const pvder_seq_norm *a, void *stream) {
    if (!ok(a)) return kEinval;
    if (a->rows == 0) return 0;                            // (the caller clears dparam)
    if (!a->h || !a->y || !a->post || !a->pre || !a->stats || !a->dh_out || !a->dy_out || (a->gate && !a->dgate_out)) return kEinval;
    if (pvder_seq_norm_workspace(a) > 0 && !a->workspace) return kEinval;
    return a->dtype == PVDER_SEQ_BF16 ? pick<__bf16>(*a, true, (hipStream_t)stream) : pick<float>(*a, true, (hipStream_t)stream);
}
