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
#include "seq_common.hpp"

namespace {

using namespace pvder_seq;

constexpr int kSumBlocks = 512;            // blocks of the backward pass that leave partial sums: two for each CU

// threads of a block: 256 where a wave holds whole rows, else one row's
constexpr int block_of(int tpr) { return tpr > 64 ? tpr : 256; }

template <typename T, int NV> struct Row {
    static constexpr int V = Vec<T>::N, E = V * NV;
    float e[E];
};

// lane t of TPR holds the vectors t, t + TPR, ...
template <typename T, int TPR, int NV> __device__ __forceinline__ void load(Row<T, NV> &r, const T *row, int t, int dim) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const typename Vec<T>::type f = load_row<T>(row, (i * TPR + t) * V, dim);
#pragma unroll
        for (int e = 0; e < V; ++e) r.e[i * V + e] = (float)f[e];
    }
}
template <typename T, int TPR, int NV> __device__ __forceinline__ void store(T *row, const Row<T, NV> &r, int t, int dim) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        typename Vec<T>::type f;
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (T)r.e[i * V + e];
        store_row<T>(row, (i * TPR + t) * V, dim, f);
    }
}
// a parameter row of fp32: `zero` behind the width
template <typename T, int TPR, int NV> __device__ __forceinline__ void load_param(Row<T, NV> &r, const float *p, int t, int dim, float otherwise) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int d = (i * TPR + t) * V + e;
            r.e[i * V + e] = d < dim ? (p ? p[d] : otherwise) : 0.f;
        }
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

// sigmoid(z) and 1 - sigmoid(z), both without cancellation
__device__ __forceinline__ void sigmoids(float z, float &s, float &c) {
    const float t = exp2f(-fabsf(z) * 1.44269504088896340736f), r = 1.f / (1.f + t);
    s = z >= 0.f ? r : t * r;
    c = z >= 0.f ? t * r : r;
    if (z != z) s = c = z;
}

template <typename T, int TPR, int NV> __global__ __launch_bounds__(block_of(TPR)) void seq_norm_forward_kernel(const pvder_seq_norm a) {
    constexpr int BLOCK = block_of(TPR), RPB = BLOCK / TPR, E = Row<T, NV>::E;
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    const int t = threadIdx.x % TPR, D = a.width;
    const long long r = blockIdx.x * (long long)RPB + threadIdx.x / TPR;
    if (TPR <= 64 && r >= a.rows) return;
    const bool on = r < a.rows;
    const int dim = on ? D : 0;
    Row<T, NV> y, h, z, w;
    load<T, TPR, NV>(y, (const T *)a.y + r * a.y_r, t, dim);
    load<T, TPR, NV>(h, (const T *)a.h + r * a.h_r, t, dim);
    if (a.gate) load<T, TPR, NV>(z, (const T *)a.gate + r * a.gate_r, t, dim);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = __builtin_fmaf(y.e[e], y.e[e], s);
    const float ry = rsqrtf(row_sum<TPR>(s, lds) / (float)D + a.eps);
    load_param<T, TPR, NV>(w, a.post, t, dim, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float u = y.e[e] * ry * w.e[e];
        if (a.gate) { float sg, c; sigmoids(z.e[e], sg, c); u *= sg; }
        y.e[e] = u;
    }
    load_param<T, TPR, NV>(w, a.scale, t, dim, 1.f);
    s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        h.e[e] = __builtin_fmaf(w.e[e], y.e[e], h.e[e]);
        s = __builtin_fmaf(h.e[e], h.e[e], s);
    }
    const float rh = rsqrtf(row_sum<TPR>(s, lds) / (float)D + a.eps);
    store<T, TPR, NV>((T *)a.h_out + r * D, h, t, dim);
    load_param<T, TPR, NV>(w, a.pre, t, dim, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) h.e[e] *= rh * w.e[e];
    store<T, TPR, NV>((T *)a.x_out + r * D, h, t, dim);
    if (on && a.stats && t == 0) { a.stats[2 * r] = ry; a.stats[2 * r + 1] = rh; }
}

template <typename T, int TPR, int NV> __global__ __launch_bounds__(block_of(TPR)) void seq_norm_backward_kernel(const pvder_seq_norm a) {
    constexpr int BLOCK = block_of(TPR), RPB = BLOCK / TPR, V = Vec<T>::N, E = Row<T, NV>::E;
    __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
    __shared__ float sums[RPB > 1 ? BLOCK * E : 1];
    const int t = threadIdx.x % TPR, D = a.width, grp = threadIdx.x / TPR;
    Row<T, NV> post, pre, scale, gpost, gpre, gscale;
    load_param<T, TPR, NV>(post, a.post, t, D, 1.f);
    load_param<T, TPR, NV>(pre, a.pre, t, D, 1.f);
    load_param<T, TPR, NV>(scale, a.scale, t, D, 1.f);
#pragma unroll
    for (int e = 0; e < E; ++e) gpost.e[e] = gpre.e[e] = gscale.e[e] = 0.f;
    const float inv = 1.f / (float)D;
    // (rows go round the blocks; every lane of a block takes as many turns: sums over more than a wave have a barrier in them)
    for (long long r0 = blockIdx.x * (long long)RPB; r0 < a.rows; r0 += gridDim.x * (long long)RPB) {
        const long long r = r0 + grp;
        const bool on = r < a.rows;
        const int dim = on ? D : 0;
        Row<T, NV> y, h, z, dh, dx;
        load<T, TPR, NV>(y, (const T *)a.y + r * a.y_r, t, dim);
        load<T, TPR, NV>(h, (const T *)a.h + r * a.h_r, t, dim);
        load<T, TPR, NV>(z, (const T *)a.gate + r * a.gate_r, t, a.gate ? dim : 0);
        load<T, TPR, NV>(dh, (const T *)a.dh + r * a.dh_r, t, a.dh ? dim : 0);
        load<T, TPR, NV>(dx, (const T *)a.dx + r * a.dx_r, t, a.dx ? dim : 0);
        const float ry = on ? a.stats[2 * r] : 0.f, rh = on ? a.stats[2 * r + 1] : 0.f;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float sg = 1.f, c = 0.f;
            if (a.gate) sigmoids(z.e[e], sg, c);
            const float u = y.e[e] * ry * post.e[e] * sg;
            h.e[e] = __builtin_fmaf(scale.e[e], u, h.e[e]);
            s = __builtin_fmaf(dx.e[e] * pre.e[e], h.e[e], s);
        }
        const float A = row_sum<TPR>(s, lds) * inv * rh * rh;
        s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float sg = 1.f, c = 0.f;
            if (a.gate) sigmoids(z.e[e], sg, c);
            const float n0 = y.e[e] * ry, n = n0 * post.e[e];
            gpre.e[e] = __builtin_fmaf(dx.e[e] * h.e[e], rh, gpre.e[e]);
            const float d = __builtin_fmaf(rh, dx.e[e] * pre.e[e] - h.e[e] * A, dh.e[e]);
            const float du = d * scale.e[e];
            gscale.e[e] = __builtin_fmaf(d, n * sg, gscale.e[e]);
            gpost.e[e] = __builtin_fmaf(du * sg, n0, gpost.e[e]);
            z.e[e] = du * n * sg * c;
            dh.e[e] = d;
            dx.e[e] = du * sg * post.e[e];
            s = __builtin_fmaf(dx.e[e], y.e[e], s);
        }
        const float B = row_sum<TPR>(s, lds) * inv * ry * ry;
#pragma unroll
        for (int e = 0; e < E; ++e) dx.e[e] = ry * (dx.e[e] - y.e[e] * B);
        store<T, TPR, NV>((T *)a.dh_out + r * D, dh, t, dim);
        store<T, TPR, NV>((T *)a.dy_out + r * D, dx, t, dim);
        if (a.gate) store<T, TPR, NV>((T *)a.dgate_out + r * D, z, t, dim);
    }
    if (!a.dparam) return;
    float *out = (gridDim.x > 1 ? a.workspace : a.dparam) + blockIdx.x * 3ll * D;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        Row<T, NV> &v = k == 0 ? gpost : (k == 1 ? gpre : gscale);
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) sums[e * BLOCK + threadIdx.x] = v.e[e];
            __syncthreads();
            if (grp == 0)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll 1
                    for (int g = 1; g < RPB; ++g) v.e[e] += sums[e * BLOCK + g * TPR + t];
        }
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int d = (i * TPR + t) * V + e;
                    if (d < D) out[k * D + d] = v.e[i * V + e];
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

struct Shape { int tpr, nv; };
// lanes to a row and vectors to a lane: the fewest lanes that hold the row at up to 16 elements a lane, 4 lanes at least
Shape shape_of(int width, int dtype) {
    const int v = dtype == PVDER_SEQ_BF16 ? 8 : 4, nv = 16 / v;
    int tpr = 4;
    while (tpr * v * nv < width) tpr <<= 1;
    return {tpr, nv};
}
int rows_per_block(int tpr) { return block_of(tpr) / tpr; }
long long sum_blocks(const pvder_seq_norm *a, int tpr) {
    const long long need = (a->rows + rows_per_block(tpr) - 1) / rows_per_block(tpr);
    return need < kSumBlocks ? need : kSumBlocks;
}

template <typename T, int TPR> int run(const pvder_seq_norm &a, bool back, hipStream_t st) {
    constexpr int NV = 16 / Vec<T>::N, BLOCK = block_of(TPR), RPB = BLOCK / TPR;
    if (back) {
        const long long blocks = sum_blocks(&a, TPR);
        seq_norm_backward_kernel<T, TPR, NV><<<dim3((unsigned)blocks), dim3(BLOCK), 0, st>>>(a);
        if (a.dparam && blocks > 1)
            seq_norm_sum_kernel<<<dim3((3 * a.width + 31) / 32), dim3(256), 0, st>>>(a.workspace, a.dparam, (int)blocks, 3 * a.width);
    } else {
        const long long blocks = (a.rows + RPB - 1) / RPB;
        if (blocks > 0x7fffffffll) return kEinval;
        seq_norm_forward_kernel<T, TPR, NV><<<dim3((unsigned)blocks), dim3(BLOCK), 0, st>>>(a);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -(int)e;
}

template <typename T> int pick(const pvder_seq_norm &a, bool back, hipStream_t st) {
    switch (shape_of(a.width, a.dtype).tpr) {
        case 4: return run<T, 4>(a, back, st);
        case 8: return run<T, 8>(a, back, st);
        case 16: return run<T, 16>(a, back, st);
        case 32: return run<T, 32>(a, back, st);
        case 64: return run<T, 64>(a, back, st);
        case 128: return run<T, 128>(a, back, st);
        case 256: return run<T, 256>(a, back, st);
        default: return run<T, 512>(a, back, st);
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
    const long long blocks = sum_blocks(a, shape_of(a->width, a->dtype).tpr);
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
