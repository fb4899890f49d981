// seq_attn.hip -- attention that decays with distance, chunk by chunk (include/pvder_sequence.h: pvder_seq_attn_run).
//
// One wave walks the tokens of one (batch row, head) and one strip of the value columns.  Its state S [dk][strip], fp32, stays
// in registers as the accumulators of the matrix cores from the first chunk to the last.  For a chunk of C tokens
//   A^T = K Q^T                          [C x C]       weights g^|x - y| on the side that x may see
//   O^T = r_x S^T Q^T + V^T P^T          [strip x C]   P = A with the weights; r_x = g^(x + 1): reach of what came before
//   S   = g^C S + K^T (w V)              [dk x strip]  w_y = g^(C - 1 - y)
// All three are computed transposed, so that the accumulators of one product already lie as the operand of the next: the row
// that a lane's accumulator r of tile t stands for is chosen (`tile_row`) so that the lane holds exactly the contraction slots
// it has to supply.  P and S never pass through LDS; K and V do, once, to be read back by columns.
//
// Bound: bytes.  A token of a head costs (2 dk + 2 dv) elements and 4 dk dv + 2 C (dk + dv) operations: with bf16, dk = dv = 64
// and C = 32 that is 48 operations per byte, where the card turns over at about 240.
#include "seq_common.hpp"

namespace {

using namespace pvder_seq;

// One wave's lanes exchange data through LDS without a barrier: its LDS operations execute in order, and this keeps the compiler
// from reordering them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- the two element types: an operand fragment is 16 bytes per lane, VPL contraction slots, KW of them over the wave ----
template <typename T> struct Ty;

template <> struct Ty<__bf16> {
    typedef b8 frag;
    static constexpr int VPL = 8, KW = 32, TT = 2, PAD = 8, PARTS = 3;
    // accumulator row mm (0..15) of tile t within a group of KW rows
    static __device__ __forceinline__ int tile_row(int t, int mm) { return 8 * (mm >> 2) + 4 * t + (mm & 3); }
    static __device__ __forceinline__ f4 mfma(frag a, frag b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // tiles t0 (, t1) of one column -> the operand that has those rows as its contraction slots
    static __device__ __forceinline__ frag operand(const f4 *t) {
        const f8 x = {t[0].x, t[0].y, t[0].z, t[0].w, t[1].x, t[1].y, t[1].z, t[1].w};
        return __builtin_convertvector(x, b8);
    }
    // w_y v_y as PARTS summands of 8 bits each: the state is an fp32 sum of fp32 products, as it would be without matrix cores
    // (one rounding to bf16 would be 2^-9 of every term and shows in the state that goes out)
    static __device__ __forceinline__ void weighted(frag v, const float *w, frag *part) {
        f8 x = __builtin_convertvector(v, f8);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= w[e];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            part[p] = __builtin_convertvector(x, b8);
            if (p + 1 < PARTS) x -= __builtin_convertvector(part[p], f8);
        }
    }
    // column fragment of an LDS tile [KW][W]: slots = rows VPL g + e, this lane's column = group base + tile_row(t, m)
    template <int W> static __device__ __forceinline__ frag column(const __bf16 *tile, int col0, int t, int m, int g) {
        const __bf16 *p = tile + (size_t)(8 * g + (m >> 2)) * (W + PAD) + col0 + 8 * (m & 3) + 4 * t;
        typedef __attribute__((address_space(3))) s4 lds4;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 4 * (W + PAD)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        const s8 r = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        return __builtin_bit_cast(b8, r);
    }
};

template <> struct Ty<float> {
    typedef f4 frag;
    static constexpr int VPL = 4, KW = 16, TT = 1, PAD = 4, PARTS = 1;
    static __device__ __forceinline__ int tile_row(int, int mm) { return mm; }
    static __device__ __forceinline__ f4 mfma(frag a, frag b, f4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ frag operand(const f4 *t) { return t[0]; }
    static __device__ __forceinline__ void weighted(frag v, const float *w, frag *part) {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[0][e] = v[e] * w[e];
    }
    template <int W> static __device__ __forceinline__ frag column(const float *tile, int col0, int, int m, int g) {
        const float *p = tile + (size_t)(4 * g) * (W + PAD) + col0 + m;
        return frag{p[0], p[W + PAD], p[2 * (W + PAD)], p[3 * (W + PAD)]};
    }
};

struct Args {
    pvder_seq_attn a;
    int seg_len, n_sib;                     // tokens of a piece; waves of one (b, h, piece): all strips of all scans
    int sib0[PVDER_SEQ_MAX_SCANS + 1];      // first wave of each scan
    long long n_groups, per_sib;            // (b, h, piece) triples; workspace floats of one wave's state
    float *carry;                           // [scan][b][h][piece]: what a piece leaves of the state before it, < 0: nothing (a start)
};

// Which (b, h, piece) and which wave of it a block is.  Blocks are dealt to the eight XCDs in turn: the waves of one triple read
// the same tensors, so they get block numbers that are 8 apart and share one L2.
__device__ __forceinline__ bool whose(const Args &A, long long &grp, int &sib) {
    const long long id = blockIdx.x, row = id / (8 * A.n_sib);
    const int in = (int)(id - row * 8 * A.n_sib);
    sib = in >> 3;
    grp = row * 8 + (in & 7);
    return grp < A.n_groups;
}

// WHOLE: heads of exactly DKP and a multiple of DVS
template <typename T, int DKP, int DVS, bool WHOLE, bool STATE_ONLY>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(DKP * DVS > 4096 ? 1 : 2)))
void seq_scan_kernel(const Args A) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int C = Y::KW, NT = C / 16, TT = Y::TT, V = Y::VPL;
    constexpr int KS = DKP / Y::KW, VS = DVS / Y::KW, NI = DKP / 16, NJ = DVS / 16;
    __shared__ __attribute__((aligned(16))) T ldsK[C * (DKP + Y::PAD)], ldsV[C * (DVS + Y::PAD)];

    long long grp;
    int sib;
    if (!whose(A, grp, sib)) return;
    int sc = 0;
    while (sc + 1 < A.a.n_scans && sib >= A.sib0[sc + 1]) ++sc;
    const pvder_seq_scan &S = A.a.scan[sc];
    const int strip = sib - A.sib0[sc], dv0 = strip * DVS;
    const int nseg = A.a.segments;
    const int seg = (int)(grp % nseg);
    const long long bh = grp / nseg;
    const int h = (int)(bh % A.a.H), b = (int)(bh / A.a.H);
    const int lane = threadIdx.x, g = lane >> 4, m = lane & 15;
    const bool rev = S.reverse != 0;
    const int DK = S.dk, DV = S.dv - dv0;                 // columns of this strip's rows that exist: dv0 .. dv0 + DV

    int len = A.a.T;
    if (A.a.lengths) { len = A.a.lengths[b]; len = len < 0 ? 0 : (len > A.a.T ? A.a.T : len); }
    const int seg_a = seg * A.seg_len;
    int seg_e = seg_a + A.seg_len;
    seg_e = seg_e > A.a.T ? A.a.T : seg_e;
    int tok_e = len < seg_e ? len : seg_e;                 // (a piece behind the last token is empty, not of negative length)
    const int tok_a = seg_a;
    tok_e = tok_e < tok_a ? tok_a : tok_e;

    const T *Q = (const T *)S.q + b * S.q_b + h * S.q_h;
    const T *K = (const T *)S.k + b * S.k_b + h * S.k_h;
    const T *Vp = (const T *)S.v + b * S.v_b + h * S.v_h + dv0;
    T *O = (T *)S.o + b * S.o_b + h * S.o_h + dv0;
    const uint8_t *St = A.a.starts ? A.a.starts + b * A.a.starts_b : nullptr;

    const float lg = log2_decay(A.a.log_decay[h]);

    // ---- the state that comes in: element (i, j, r) is S[KW (i / TT) + tile_row(i % TT, 4 g + r)][KW (j / TT) + tile_row(j % TT, m)]
    f4 s[NI][NJ];
    const bool first = rev ? seg == nseg - 1 : seg == 0;
    float *ws = A.a.workspace ? A.a.workspace + ((grp * A.n_sib + sib) * A.per_sib) + lane * 4 : nullptr;
    if (!STATE_ONLY && nseg > 1) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[i][j] = *(const f4 *)(ws + (i * NJ + j) * 256);
    } else if (!STATE_ONLY && first && S.s_in) {
        const float *p = S.s_in + b * S.s_b + h * S.s_h;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = Y::KW * (i / TT) + Y::tile_row(i % TT, 4 * g + r), dv = Y::KW * (j / TT) + Y::tile_row(j % TT, m);
                    s[i][j][r] = dk < DK && dv < DV ? p[dk * S.s_k + (dv0 + dv) * S.s_v] : 0.f;
                }
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- weights that depend on the head alone, and those that depend on the chunk's length
    float dw[NT][TT][4], wy[V], rx[NT], gn = 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int x = 16 * nt + m, y = V * g + 4 * t + r, d = rev ? y - x : x - y;
                dw[nt][t][r] = d >= 0 ? S.a_intra * power(lg, d) : 0.f;
            }
    int n_have = 0;
    auto by_length = [&](int n) {
        if (n == n_have) return;
        n_have = n;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int y = V * g + e, d = rev ? y + 1 : n - 1 - y;
            wy[e] = y < n ? S.a_write * power(lg, d) : 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int x = 16 * nt + m, d = rev ? n - 1 - x : x + 1;
            rx[nt] = x < n ? S.a_read * power(lg, d) : 0.f;
        }
        gn = power(lg, n);
    };

    // ---- loads of a chunk [a, a + n), raw: rows behind n and pieces behind the head's end are read from places that exist, and put
    // right by `mend` when they are used.  Offsets of a lane are 32-bit, from a base that the wave shares.
    frag nq[NT][KS], nk[TT][KS], nv[TT][VS];
    const unsigned q_t = (unsigned)(S.q_t * sizeof(T)), k_t = (unsigned)(S.k_t * sizeof(T)), v_t = (unsigned)(S.v_t * sizeof(T));
    const unsigned in_row = V * g * sizeof(T);
    unsigned qo[NT], ko[TT], vo[TT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) qo[nt] = (16 * nt + m) * q_t;
#pragma unroll
    for (int t = 0; t < TT; ++t) { ko[t] = Y::tile_row(t, m) * k_t; vo[t] = Y::tile_row(t, m) * v_t; }
    auto piece = [&](const char *base, unsigned row, int p, int dim) {
        frag f;
        if constexpr (WHOLE) {
            __builtin_memcpy(&f, base + (row + in_row) + p * (int)(Y::KW * sizeof(T)), 16);
        } else if (dim >= V) {
            const int d = p * Y::KW + V * g, last = dim - V;
            __builtin_memcpy(&f, base + (row + (unsigned)((d < last ? d : last) * sizeof(T))), 16);
        } else {                                            // heads of a few elements
            const T *r = (const T *)(base + row);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = r[e < dim ? e : 0];
        }
        return f;
    };
    auto mend = [&](frag &f, bool row_is, int p, int dim) {
        if constexpr (!WHOLE) {
            const int d = p * Y::KW + V * g, last = dim - V;
            if (dim % V != 0) {
                if (dim >= V) f = behind(f, d > last ? d - last : 0);
                else
#pragma unroll
                    for (int e = 0; e < V; ++e) f[e] = d + e < dim ? f[e] : (T)0.f;
            }
            row_is = row_is && d < dim;
        }
        const u4 u = __builtin_bit_cast(u4, f);
        f = __builtin_bit_cast(frag, row_is ? u : u4{0u, 0u, 0u, 0u});
    };
    auto load_q = [&](int a, int n) {
        if constexpr (!STATE_ONLY) {
            const char *base = (const char *)(Q + (long long)a * S.q_t);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) nq[nt][ks] = piece(base, 16 * nt + m < n ? qo[nt] : 0u, ks, DK);
        }
    };
    auto load_kv = [&](int a, int n) {
        const char *kb = (const char *)(K + (long long)a * S.k_t), *vb = (const char *)(Vp + (long long)a * S.v_t);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const bool is = Y::tile_row(t, m) < n;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) nk[t][ks] = piece(kb, is ? ko[t] : 0u, ks, DK);
#pragma unroll
            for (int vs = 0; vs < VS; ++vs) nv[t][vs] = piece(vb, is ? vo[t] : 0u, vs, DV);
        }
    };
    auto mend_all = [&](int n) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if constexpr (!STATE_ONLY) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mend(nq[nt][ks], 16 * nt + m < n, ks, DK);
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) mend(nk[t][ks], Y::tile_row(t, m) < n, ks, DK);
        }
#pragma unroll
        for (int vs = 0; vs < VS; ++vs)
#pragma unroll
            for (int t = 0; t < TT; ++t) mend(nv[t][vs], Y::tile_row(t, m) < n, vs, DV);
    };
    uint8_t nflag = 0;
    auto load_flags = [&](int a, int n) { nflag = St && lane < n ? St[(long long)(a + lane) * A.a.starts_t] : 0; };

    bool any_start = false;
    int pos = rev ? tok_e : tok_a, most = C;
    auto left = [&]() { const int l = rev ? pos - tok_a : tok_e - pos; return l < most ? l : most; };
    int n = left();
    if (n > 0) { const int a = rev ? pos - n : pos; load_kv(a, n); load_q(a, n); load_flags(a, n); }
    while (n > 0) {
        by_length(n);
        const int a = rev ? pos - n : pos, pos0 = pos;
        const unsigned mask = St ? (unsigned)__ballot(nflag != 0) : 0u;
        // (the starts of a chunk as bits: x and y are of one episode if no bit lies behind the earlier and up to the later)
        const unsigned upto_last = (2u << (n - 1)) - 1u;
        if (!WHOLE || n < C) mend_all(n);
        wave_sync();                                     // the chunk before has been read
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int y = Y::tile_row(t, m);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) *(frag *)(ldsK + y * (DKP + Y::PAD) + ks * Y::KW + V * g) = nk[t][ks];
#pragma unroll
            for (int vs = 0; vs < VS; ++vs) *(frag *)(ldsV + y * (DVS + Y::PAD) + vs * Y::KW + V * g) = nv[t][vs];
        }
        wave_sync();
        // A value that is not finite would reach other tokens through a weight of zero (0 x NaN).  Such a chunk is taken token by
        // token instead, where no token shares a product with another.  The check sums the operands on the matrix cores.
        float z = 0.f;
        if constexpr (TT == 2) {
            f4 z0 = {0.f, 0.f, 0.f, 0.f}, z1 = z0;
            frag one;
#pragma unroll
            for (int e = 0; e < V; ++e) one[e] = (T)1.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) { z0 = Y::mfma(one, nk[0][ks], z0); z1 = Y::mfma(one, nk[1][ks], z1); }
#pragma unroll
            for (int vs = 0; vs < VS; ++vs) { z0 = Y::mfma(one, nv[0][vs], z0); z1 = Y::mfma(one, nv[1][vs], z1); }
            z = z0[0] * 0.f + z1[0] * 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) z = __builtin_fmaf((float)nk[0][ks][e], 0.f, z);
#pragma unroll
                for (int vs = 0; vs < VS; ++vs) z = __builtin_fmaf((float)nv[0][vs][e], 0.f, z);
            }
        }
        frag p[NT];
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                f4 at[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    at[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) at[t] = Y::mfma(nk[t][ks], nq[nt][ks], at[t]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float w = dw[nt][t][r];
                        if (mask) {
                            const int x = 16 * nt + m, y = V * g + 4 * t + r;
                            const unsigned bits = ((2u << x) - 1u) ^ ((2u << y) - 1u);   // the tokens behind one, up to the other
                            w = (mask & bits) == 0 ? w : 0.f;
                        }
                        at[t][r] = mul_or_zero(at[t][r], w);
                    }
                }
                p[nt] = Y::operand(at);
            }
        }
        frag vf[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) vf[j] = Y::template column<DVS>(ldsV, Y::KW * (j / TT), j % TT, m, g);
        // the next chunk's loads are in flight while this one is computed
        pos += rev ? -n : n;
        most = C;
        const int n2 = left(), a2 = rev ? pos - n2 : pos;
        if (n2 > 0) load_kv(a2, n2);
        f4 o[VS][NT][TT];
        if constexpr (!STATE_ONLY) {
            // P and S as operands are rounded to the inputs' type: 2^-9 of each term at bf16, as much as the output's own rounding; the
            // sums are fp32
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) o[j / TT][nt][j % TT] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    f4 rows[TT];
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) rows[tt] = s[ks * TT + tt][j];
                    const frag sf = Y::operand(rows);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[j / TT][nt][j % TT] = Y::mfma(sf, nq[nt][ks], o[j / TT][nt][j % TT]);
                }
            }
        }
        if (n2 > 0) { load_q(a2, n2); load_flags(a2, n2); }
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float reach = rx[nt];
                if (mask) {
                    const unsigned upto = (2u << (16 * nt + m)) - 1u;
                    reach = (rev ? mask & upto_last & ~upto : mask & upto) == 0 ? reach : 0.f;
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    f4 &t = o[j / TT][nt][j % TT];
#pragma unroll
                    for (int r = 0; r < 4; ++r) t[r] = mul_or_zero(t[r], reach);
                    t = Y::mfma(vf[j], p[nt], t);
                }
            }
        }
        if (n > 1 && __any(z != 0.f || z != z)) {
            pos = pos0;
            most = n = 1;
            const int a1 = rev ? pos - 1 : pos;
            load_kv(a1, 1); load_q(a1, 1); load_flags(a1, 1);
            continue;
        }
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int x = 16 * nt + m;
                if (x < n) {
                    T *row = O + (long long)(a + x) * S.o_t;
#pragma unroll
                    for (int jg = 0; jg < VS; ++jg) {
                        const frag f = Y::operand(o[jg][nt]);
                        if constexpr (WHOLE) __builtin_memcpy(row + jg * Y::KW + V * g, &f, 16);
                        else store_row<T>(row, jg * Y::KW + V * g, DV, f);
                    }
                }
            }
        }
        // ---- the state behind the chunk
        float w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = wy[e];
            if (mask) {
                const unsigned upto = (2u << ((V * g + e) & 31)) - 1u;
                if ((rev ? mask & upto : mask & upto_last & ~upto) != 0) w[e] = 0.f;
            }
        }
        const bool fresh = (mask & upto_last) != 0;
        any_start = any_start || fresh;
        const float gs = fresh ? 0.f : gn;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][j][r] = mul_or_zero(s[i][j][r], gs);
        frag kt[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) kt[i] = Y::template column<DKP>(ldsK, Y::KW * (i / TT), i % TT, m, g);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            frag part[Y::PARTS];
            Y::weighted(vf[j], w, part);
#pragma unroll
            for (int pp = 0; pp < Y::PARTS; ++pp)
#pragma unroll
                for (int i = 0; i < NI; ++i) s[i][j] = Y::mfma(kt[i], part[pp], s[i][j]);
        }
        n = n2;
    }

    if constexpr (STATE_ONLY) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) *(f4 *)(ws + (i * NJ + j) * 256) = s[i][j];
        if (lane == 0 && strip == 0)
            A.carry[((long long)sc * A.a.B * A.a.H + bh) * nseg + seg] = any_start ? -1.f : power(lg, tok_e - tok_a);
    } else {
        // rows at and behind the length
        for (int t = tok_e + g; t < seg_e; t += 4)
#pragma unroll
            for (int jg = 0; jg < VS; ++jg)
#pragma unroll
                for (int u = m; u < Y::KW / V; u += 16) {
                    frag z;
#pragma unroll
                    for (int e = 0; e < V; ++e) z[e] = (T)0.f;
                    store_row<T>(O + (long long)t * S.o_t, jg * Y::KW + V * u, DV, z);
                }
        if ((rev ? seg == 0 : seg == nseg - 1) && S.s_out) {
            float *p = S.s_out + b * S.s_b + h * S.s_h;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int dk = Y::KW * (i / TT) + Y::tile_row(i % TT, 4 * g + r), dv = Y::KW * (j / TT) + Y::tile_row(j % TT, m);
                        if (dk < DK && dv < DV) p[dk * S.s_k + (dv0 + dv) * S.s_v] = s[i][j][r];
                    }
        }
    }
}

// The states that come into the pieces, from what each piece adds: s_(i+1) = carry_i s_i + u_i, written over u_i as s_i.
template <typename T, int DKP, int DVS> __global__ __launch_bounds__(256) void seq_join_kernel(const Args A) {
    typedef Ty<T> Y;
    constexpr int Q = DKP * DVS / 4, TT = Y::TT, NJ = DVS / 16;
    const int nseg = A.a.segments;
    const long long id = blockIdx.x * 256ll + threadIdx.x, wave = id / Q;
    const int at = (int)(id - wave * Q);
    if (wave >= (long long)A.a.B * A.a.H * A.n_sib) return;
    const int sib = (int)(wave % A.n_sib);
    const long long bh = wave / A.n_sib;
    int sc = 0;
    while (sc + 1 < A.a.n_scans && sib >= A.sib0[sc + 1]) ++sc;
    const pvder_seq_scan &S = A.a.scan[sc];
    const int h = (int)(bh % A.a.H), b = (int)(bh / A.a.H);
    const bool rev = S.reverse != 0;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (S.s_in) {
        const int tile = at >> 6, lane = at & 63, g = lane >> 4, m = lane & 15, i = tile / NJ, j = tile % NJ;
        const int dv = (sib - A.sib0[sc]) * DVS + Y::KW * (j / TT) + Y::tile_row(j % TT, m);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int dk = Y::KW * (i / TT) + Y::tile_row(i % TT, 4 * g + r);
            if (dk < S.dk && dv < S.dv) s[r] = S.s_in[b * S.s_b + h * S.s_h + dk * S.s_k + dv * S.s_v];
        }
    }
    const float *carry = A.carry + ((long long)sc * A.a.B * A.a.H + bh) * nseg;
    float *ws = A.a.workspace + at * 4;
    for (int n = 0; n < nseg; ++n) {
        const int seg = rev ? nseg - 1 - n : n;
        f4 *p = (f4 *)(ws + ((bh * nseg + seg) * A.n_sib + sib) * A.per_sib);
        const f4 u = *p;
        const float c = carry[seg];
        *p = s;
        s = c < 0.f ? u : s * c + u;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
int padded(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

// One kernel per pair of padded sizes.  The state of a wave is dkp x dvs: 64 x 64 at most, 128 x 32 where dk needs 128.
struct Plan { int dkp, dvs, n_sib, sib0[PVDER_SEQ_MAX_SCANS + 1]; };

bool plan_of(const pvder_seq_attn *a, Plan &P) {
    if (!a || a->n_scans < 1 || a->n_scans > PVDER_SEQ_MAX_SCANS || a->B < 0 || a->T < 0 || a->H < 1) return false;
    if (a->dtype != PVDER_SEQ_F32 && a->dtype != PVDER_SEQ_BF16) return false;
    int dk = 0, dv = 0;
    for (int i = 0; i < a->n_scans; ++i) {
        const pvder_seq_scan &s = a->scan[i];
        if (s.dk < 1 || s.dv < 1 || s.dk > PVDER_SEQ_MAX_HEAD || s.dv > PVDER_SEQ_MAX_HEAD) return false;
        dk = s.dk > dk ? s.dk : dk;
        dv = s.dv > dv ? s.dv : dv;
    }
    P.dkp = padded(dk);
    P.dvs = padded(dv);
    if (P.dvs > 64) P.dvs = 64;
    if (P.dkp == 128) P.dvs = 32;
    P.n_sib = 0;
    for (int i = 0; i < a->n_scans; ++i) {
        P.sib0[i] = P.n_sib;
        P.n_sib += (a->scan[i].dv + P.dvs - 1) / P.dvs;
    }
    for (int i = a->n_scans; i <= PVDER_SEQ_MAX_SCANS; ++i) P.sib0[i] = P.n_sib;
    return true;
}

int seg_len_of(const pvder_seq_attn *a) {
    const int c = 32, per = (a->T + a->segments - 1) / a->segments;
    return (per + c - 1) / c * c;
}

template <typename T, int DKP, int DVS, bool WHOLE> int launch(const Args &A, hipStream_t st) {
    const long long blocks = (A.n_groups + 7) / 8 * 8 * A.n_sib;
    if (blocks > 0x7fffffffll) return kEinval;
    if (A.a.segments > 1) {
        seq_scan_kernel<T, DKP, DVS, WHOLE, true><<<dim3((unsigned)blocks), dim3(64), 0, st>>>(A);
        const long long items = (long long)A.a.B * A.a.H * A.n_sib * (DKP * DVS / 4);
        seq_join_kernel<T, DKP, DVS><<<dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st>>>(A);
    }
    seq_scan_kernel<T, DKP, DVS, WHOLE, false><<<dim3((unsigned)blocks), dim3(64), 0, st>>>(A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -(int)e;
}

template <typename T, int DKP, int DVS> int fit(const Args &A, hipStream_t st) {
    bool whole = true;
    for (int i = 0; i < A.a.n_scans; ++i) whole = whole && A.a.scan[i].dk == DKP && A.a.scan[i].dv % DVS == 0;
    return whole ? launch<T, DKP, DVS, true>(A, st) : launch<T, DKP, DVS, false>(A, st);
}

template <typename T> int pick(const Args &A, const Plan &P, hipStream_t st) {
    if (P.dkp == 32) return P.dvs == 32 ? fit<T, 32, 32>(A, st) : fit<T, 32, 64>(A, st);
    if (P.dkp == 64) return P.dvs == 32 ? fit<T, 64, 32>(A, st) : fit<T, 64, 64>(A, st);
    return fit<T, 128, 32>(A, st);
}

}  // namespace

extern "C" int64_t pvder_seq_attn_plan(pvder_seq_attn *a) {
    Plan P;
    if (!plan_of(a, P)) return kEinval;
    const long long waves = (long long)a->B * a->H * P.n_sib;
    a->segments = 1;
    if (waves >= 1 && a->T >= 256) {
        const long long want = 2048 / waves, most = a->T / 128;
        const long long n = want < most ? want : most;
        a->segments = n < 2 ? 1 : (int32_t)n;
    }
    if (a->segments == 1) return 0;
    const int64_t bhs = (int64_t)a->B * a->H * a->segments;
    return bhs * P.n_sib * P.dkp * P.dvs + bhs * a->n_scans;
}

extern "C" int pvder_seq_attn_run(const pvder_seq_attn *a, void *stream) {
    Args A;
    Plan P;
    if (!plan_of(a, P) || a->segments < 1 || !a->log_decay) return kEinval;
    if (a->segments > 1 && (!a->workspace || ((uintptr_t)a->workspace & 15))) return kEinval;
    if (a->B > 0 && a->T > 0)
        for (int i = 0; i < a->n_scans; ++i)
        {
            const pvder_seq_scan &s = a->scan[i];
            if (!s.q || !s.k || !s.v || !s.o) return kEinval;
            const int64_t most = PVDER_SEQ_MAX_TOKEN_STRIDE / (a->dtype == PVDER_SEQ_BF16 ? 2 : 4);
            if (s.q_t < 0 || s.k_t < 0 || s.v_t < 0 || s.q_t > most || s.k_t > most || s.v_t > most) return kEinval;
        }
    if (a->B == 0) return 0;
    A.a = *a;
    if (A.a.T == 0) A.a.segments = 1;
    A.seg_len = A.a.T ? seg_len_of(&A.a) : 32;
    A.n_sib = P.n_sib;
    for (int i = 0; i <= PVDER_SEQ_MAX_SCANS; ++i) A.sib0[i] = P.sib0[i];
    A.n_groups = (long long)a->B * a->H * A.a.segments;
    A.per_sib = (long long)P.dkp * P.dvs;
    A.carry = A.a.segments > 1 ? A.a.workspace + A.n_groups * P.n_sib * A.per_sib : nullptr;
    return a->dtype == PVDER_SEQ_BF16 ? pick<__bf16>(A, P, (hipStream_t)stream) : pick<float>(A, P, (hipStream_t)stream);
}
