// seq_attn.hip -- attention that decays with distance, chunk by chunk (include/pvder_sequence.h: pvder_seq_attn_run).
//
// One wave walks the tokens of one (batch row, head) and one strip of the value columns.  Its state S [dk][strip], fp32, stays
// in registers as the accumulators of the matrix cores from the first chunk to the last.  For a chunk of C tokens
//   A^T = K Q^T                          [C x C]       weights g^|x - y| on the side that x may see
//   O^T = r_x S^T Q^T + V^T P^T          [strip x C]   P = A with the weights; r_x = g^(x + 1): reach of what came before
//   S   = g^C S + K^T (w V)              [dk x strip]  w_y = g^(C - 1 - y)
// All three are computed transposed, so that the accumulators of one product already lie as the operand of the next: the row
// that a lane's accumulator r of tile t stands for is chosen (`tile_row`) so that the lane holds exactly the contraction slots
// it has to supply.  P and S stay in registers.  Q, K and V come in whole lines, one chunk ahead, and pass through LDS, to be read
// by rows (Q, K) and by columns (K, V); the output goes through the place of Q, to leave in whole lines too.
//
// Long T with few heads is cut into pieces that run side by side, in three launches: what each piece adds to the state
// (`STATE_ONLY`), the states that come into the pieces (seq_join_kernel), and the outputs.  The three gradients are scans too; of
// their piece states the backward pass works out one, that of dv: dk's is its transpose, dq's the transpose of the forward pass's.
//
// Bound: bytes.  A token of a head costs (2 dk + 2 dv) elements and (2 + 2 p) dk dv + 2 C (dk + dv) operations, p the summands of w V
// (`weighted`): with bf16, dk = dv = 64 and C = 32 that is 64 operations per byte for p = 2, 80 for p = 3, and 8 more for the check that K
// and V are finite, where the card turns over at about 240.  fp32 has p = 1, C = 16 and matrix instructions of an eighth of the rate: 20
// operations per byte of the 30 at which it turns over.
//
// Measured, time of the kernels and share of 5.2 TB/s for each tensor once: forward 128 windows of 2048 tokens x 16 heads of 64,
// bf16, 489 us, 85 %; 1024 tokens, fp32, 476 us, 86 %; heads of 128, bf16, 64 x 1024 x 16, 300-316 us, 65-69 % (the state fills the
// registers and each strip of 32 columns reads Q and K again); heads of 32, 512 x 1024 x 8, 260 us, 79 %.  In pieces: one stream of
// 16384 tokens x 8 heads of 128, bf16, 96 us, 27 % (states 27, join 18, outputs 51); forward and backward, 4 x 4096 x 16 heads of 64,
// bf16, 170 us, 31 %.  Windows of 160 x 4 heads of 64, 64 of them, fp32, forward and backward, 61 us, 20 % (latency: ten chunks, one
// behind the other).
#include "seq_common.hpp"

namespace {

using namespace pvder_seq;

// One wave's lanes exchange data through LDS without a barrier: its LDS operations execute in order, and this keeps the compiler
// from reordering them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The parts of a chunk's work are scheduled by themselves: mixed, their operands do not fit the registers
__device__ __forceinline__ void phase() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The value as it is at this place: keeps what a rare branch computes from it out of the registers of the whole loop
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// ---- the two element types: an operand fragment is 16 bytes per lane, VPL contraction slots, KW of them over the wave ----
template <typename T> struct Ty;

template <> struct Ty<__bf16> {
    typedef b8 frag;
    static constexpr int VPL = 8, KW = 32, TT = 2;
    // LDS tiles, rows of W elements in pieces of 16 bytes.  Tiles that are read by columns (4 rows of 64 bytes together) have rows 64
    // bytes apart in the 256 bytes of the banks, those that are read by rows (a piece of 8 rows together) 16.  All places of a lane are
    // one register and constants.
    static constexpr int row(int w) { return w == 32 ? 32 : w + 32; }
    static constexpr int size(int w) { return KW * row(w); }
    // (128 wide they are turned instead: with the 16 bytes eight waves of a CU would not find room in its LDS)
    static constexpr int size_rows(int w) { return KW * (w == 128 ? w : w + 8); }
    template <int W> static __device__ __forceinline__ int at(int r, int piece) { return r * row(W) + 8 * piece; }
    template <int W> static __device__ __forceinline__ int at_rows(int r, int piece) { return W == 128 ? r * W + 8 * (piece ^ (r & 7)) : r * (W + 8) + 8 * piece; }
    // accumulator row mm (0..15) of tile t within a group of KW rows
    static __device__ __forceinline__ int tile_row(int t, int mm) { return 8 * (mm >> 2) + 4 * t + (mm & 3); }
    static __device__ __forceinline__ f4 mfma(frag a, frag b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // tiles t0 (, t1) of one column -> the operand that has those rows as its contraction slots
    static __device__ __forceinline__ frag operand(const f4 *t) {
        const f8 x = {t[0].x, t[0].y, t[0].z, t[0].w, t[1].x, t[1].y, t[1].z, t[1].w};
        return __builtin_convertvector(x, b8);
    }
    // w_y v_y as P summands of 8 bits each, P - 1 of them below the first: three are fp32's 24 bits, so a state that is returned is an fp32
    // sum of fp32 products; two (off by 2^-16 of each term at most) where only outputs of 8 bits are made of it.  One (2^-8) would show there
    // too.
    template <int P> static __device__ __forceinline__ void weighted(frag v, const float *w, frag *part) {
        f8 x = __builtin_convertvector(v, f8);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= w[e];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            part[p] = __builtin_convertvector(x, b8);
            if (p + 1 < P) x -= __builtin_convertvector(part[p], f8);
        }
    }
    // column fragment of an LDS tile [KW][W]: slots = rows VPL g + e, this lane's column = 32 (j / 2) + tile_row(j % 2, m)
    template <int W> static __device__ __forceinline__ frag column(const __bf16 *tile, int j, int m, int g) {
        const __bf16 *p = tile + at<W>(8 * g + (m >> 2), 4 * (j >> 1) + (m & 3)) + 4 * (j & 1);
        typedef __attribute__((address_space(3))) s4 lds4;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 4 * row(W)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        const s8 r = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        return __builtin_bit_cast(b8, r);
    }
};

template <> struct Ty<float> {
    typedef f4 frag;
    static constexpr int VPL = 4, KW = 16, TT = 1;
    static constexpr int size(int w) { return KW * (w + 4); }
    static constexpr int size_rows(int w) { return KW * (w + 4); }
    template <int W> static __device__ __forceinline__ int at(int row, int piece) { return row * (W + 4) + 4 * piece; }
    template <int W> static __device__ __forceinline__ int at_rows(int row, int piece) { return row * (W + 4) + 4 * piece; }
    static __device__ __forceinline__ int tile_row(int, int mm) { return mm; }
    static __device__ __forceinline__ f4 mfma(frag a, frag b, f4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ frag operand(const f4 *t) { return t[0]; }
    template <int> static __device__ __forceinline__ void weighted(frag v, const float *w, frag *part) {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[0][e] = v[e] * w[e];
    }
    template <int W> static __device__ __forceinline__ frag column(const float *tile, int j, int m, int g) {
        const float *p = tile + 4 * g * (W + 4) + 16 * j + m;
        return frag{p[0], p[W + 4], p[2 * (W + 4)], p[3 * (W + 4)]};
    }
};

// LDS of a wave: a chunk's rows of Q, K and V
template <typename T> constexpr int tile_bytes(int dkp, int dvs) { return (Ty<T>::size(dkp) + Ty<T>::size(dvs) + Ty<T>::size_rows(dkp > dvs ? dkp : dvs)) * (int)sizeof(T); }

// Where the states that come into a scan's pieces lie: as the wave that made them held them, tile by tile, a strip of `side` tiles beside each
// other after the other.  They may be of another scan, whose k is this one's v and whose v is its k: transposed then.
struct States {
    const float *at;                        // of the first (b, h, piece); `piece` floats further the next
    long long piece;
    int side_log2, strips, tiles;           // tiles of dk
    bool transposed;
};

struct Args {
    pvder_seq_attn a;
    int seg_len, n_sib;                     // tokens of a piece; strips of one (b, h, piece), all scans together
    int sib0[PVDER_SEQ_MAX_SCANS + 1];      // first strip of each scan
    unsigned n_groups;                      // (b, h, piece) triples
    unsigned together_log2;                 // how many of them on end belong to one XCD
    long long per_sib;                      // state pass and join: workspace floats of one strip's state
    float *carry;                           // [scan][b][h][piece]: what a piece leaves of the state before it (0 behind a start)
    States states[PVDER_SEQ_MAX_SCANS];     // main pass, several pieces
};

// Which (b, h, piece) a block is of, and which of its strips, all scans together.  Blocks are dealt to the eight XCDs in turn: the strips
// of one triple read the same tensors, so they get block numbers that are 8 apart and share one L2.  So do four triples on end where that
// pays (`fours`).
__device__ __forceinline__ bool whose(const Args &A, unsigned &grp, int &sib) {
    const unsigned row = (blockIdx.x >> 3) / (unsigned)A.n_sib;
    sib = (int)((blockIdx.x >> 3) - row * (unsigned)A.n_sib);
    const unsigned t = (1u << A.together_log2) - 1u;
    grp = ((((row >> A.together_log2) * 8 + (blockIdx.x & 7)) << A.together_log2) + (row & t));
    return grp < A.n_groups;
}

// A block is one wave: one strip of one scan over one (b, h, piece).  Strips of a head in one block, on one CU, were up to twice as slow
// (128 x 128, 160 tokens: 23 us against 12): four waves that walk in step ask the CU's L1 and LDS for the same at the same time.
// WHOLE: heads of exactly DKP and a multiple of DVS.  STATE_ONLY: only the state behind a piece is wanted.  PARTS: see `weighted`.
template <typename T, int DKP, int DVS, bool WHOLE, bool STATE_ONLY, int PARTS>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void seq_scan_kernel(const Args A) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int C = Y::KW, NT = C / 16, TT = Y::TT, V = Y::VPL;
    constexpr int KS = DKP / Y::KW, VS = DVS / Y::KW, NI = DKP / 16, NJ = DVS / 16;
    // bf16 heads of 128, and ragged ones of 64: the weights within a chunk are worked out again for each.  Held, they go to scratch memory,
    // and a wait for one that comes back is a wait for the next chunk's loads, too (64 x 1024 x 16 heads of 128: 375 us, 308-346 so; 128 x 1024 x
    // 16 heads of 60: 351 and 317; whole ones of 64 find room: training, 64 x 512 x 16, 190 and 197)
    constexpr bool AGAIN = TT == 2 && !STATE_ONLY && (DKP == 128 || (!WHOLE && DKP * DVS >= 4096));
    extern __shared__ __attribute__((aligned(16))) char lds[];

    unsigned grp;
    int sib, sc = 0;
    if (!whose(A, grp, sib)) return;
    while (sc + 1 < A.a.n_scans && sib >= A.sib0[sc + 1]) ++sc;
    const pvder_seq_scan &S = A.a.scan[sc];
    const int strip = sib - A.sib0[sc], dv0 = strip * DVS;
    T *ldsK = (T *)lds, *ldsV = ldsK + Y::size(DKP), *ldsQ = ldsV + Y::size(DVS);       // (ldsQ takes the output when Q has been read)
    const int nseg = A.a.segments;
    const unsigned bh = nseg == 1 ? grp : grp / (unsigned)nseg;
    const int seg = (int)(grp - bh * (unsigned)nseg), b = (int)(bh / (unsigned)A.a.H), h = (int)(bh - (unsigned)b * (unsigned)A.a.H);
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const bool rev = S.reverse != 0;
    const int DK = S.dk, DV = S.dv - dv0;                 // columns of this strip that exist, and of those behind it

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
    const T *Vp = (const T *)S.v + b * S.v_b + h * S.v_h;
    T *O = (T *)S.o + b * S.o_b + h * S.o_h;
    const uint8_t *St = A.a.starts ? A.a.starts + b * A.a.starts_b : nullptr;

    const float lg = log2_decay(A.a.log_decay[h]);

    // ---- the state that comes in: element (i, j, r) is S[KW (i / TT) + tile_row(i % TT, 4 g + r)][KW (j / TT) + tile_row(j % TT, m)]
    f4 s[NI][NJ];
    auto state_elements = [&](auto &&f) {                   // f(i, j, r, whether the head has the element, its offset in bytes)
        const int g4 = 4 * (here(lane) >> 4), mm = here(lane) & 15;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = Y::KW * (i / TT) + Y::tile_row(i % TT, g4 + r), dv = Y::KW * (j / TT) + Y::tile_row(j % TT, mm);
                    f(i, j, r, dk < DK && dv < DV, (unsigned)dk * (unsigned)(4 * S.s_k) + (unsigned)(dv0 + dv) * (unsigned)(4 * S.s_v));
                }
    };
    const bool first = rev ? seg == nseg - 1 : seg == 0;
    if (!STATE_ONLY && nseg > 1) {
        const States &W = A.states[sc];
        const gbytes p = shared_base(W.at + grp * W.piece);
        const int across = (16 * (m >> 2) + 4 * g) * 16 + 4 * (m & 3);      // element (m, 4 g) of a tile
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int si = W.transposed ? strip * NJ + j : i, sj = W.transposed ? i : strip * NJ + j, of = sj >> W.side_log2;
                const unsigned tile = (unsigned)((((of * W.tiles + si) << W.side_log2) + (sj & ((1 << W.side_log2) - 1))) * 1024);
                s[i][j] = f4{0.f, 0.f, 0.f, 0.f};
                if (si < W.tiles && of < W.strips) {        // (what is padded further here than there is zero)
                    if (!W.transposed) s[i][j] = *(const __attribute__((address_space(1))) f4 *)(p + tile + lane * 16);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][j][r] = *(const __attribute__((address_space(1))) float *)(p + tile + across + 16 * r);
                }
            }
    } else if (!STATE_ONLY && first && S.s_in) {
        const gbytes p = shared_base(S.s_in + b * S.s_b + h * S.s_h);
        state_elements([&](int i, int j, int r, bool is, unsigned at) {
            const float x = *(const __attribute__((address_space(1))) float *)(p + (is ? at : 0u));
            s[i][j][r] = is ? x : 0.f;
        });
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- weights that depend on the head alone, and those that depend on the chunk's length
    float dw[NT][TT][4], wy[V], rx[NT], gn = 1.f;
    auto within = [&](int g, int m) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int x = 16 * nt + m, y = V * g + 4 * t + r, d = rev ? y - x : x - y;
                    const float w = S.a_intra * power(lg, d);
                    dw[nt][t][r] = d >= 0 ? w : 0.f;
                }
    };
    if constexpr (!AGAIN) within(g, m);
    int n_have = 0;
    auto by_length = [&](int n) {
        if (n == n_have) return;
        n_have = n;
        const int g = here(lane) >> 4, m = here(lane) & 15;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int y = V * g + e, d = rev ? y + 1 : n - 1 - y;
            const float w = S.a_write * power(lg, d);
            wy[e] = y < n ? w : 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int x = 16 * nt + m, d = rev ? n - 1 - x : x + 1;
            const float w = S.a_read * power(lg, d);
            rx[nt] = x < n ? w : 0.f;
        }
        gn = power(lg, n);
    };

    // ---- loads of a chunk [a, a + n): rows behind n and pieces behind the head's end are outside of the window and read as zeros; the
    // piece that the head's end cuts is read from 16 bytes before that end, and shifted by `mend` when it is used.  Neighbouring lanes
    // take neighbouring pieces of a row: the L1 serves a line a cycle, and in the operands' own order, a row a lane, it served four times
    // as many.
    constexpr int PK = DKP / V, RK = 64 / PK, NK = C / RK;  // pieces of a row of K, rows that a load takes, loads
    constexpr int PV = DVS / V, RV = 64 / PV, NV = C / RV;
    constexpr int KP = Y::KW / V;                           // pieces of a group of contraction slots: four
    frag sq[NK], sk[NK], sv[NV];
    const unsigned q_t = (unsigned)(S.q_t * sizeof(T)), k_t = (unsigned)(S.k_t * sizeof(T)), v_t = (unsigned)(S.v_t * sizeof(T));
    const unsigned o_t = (unsigned)(S.o_t * sizeof(T));
    const unsigned row_k = DK * sizeof(T), row_v = S.dv * sizeof(T);
    const int rk = lane / PK, pk = lane % PK, rv = lane / PV, pv = lane % PV;
    constexpr unsigned OUTSIDE = 0x80000000u;               // of every window, whatever rows are added
    auto in_row = [&](int d, int dim) {                     // the bytes of elements d .. d + V of a row of dim
        if (!WHOLE && d >= dim) return OUTSIDE;
        return (unsigned)((WHOLE || d <= dim - V ? d : dim - V) * sizeof(T));
    };
    const int dk0 = pk * V, dvp = dv0 + pv * V;             // the first elements of a lane's pieces
    const unsigned qo = rk * q_t + in_row(dk0, DK), ko = rk * k_t + in_row(dk0, DK), vo = rv * v_t + in_row(dvp, S.dv);
    auto piece = [&](window w, unsigned off) { return __builtin_bit_cast(frag, __builtin_amdgcn_raw_buffer_load_b128(w, off, 0, 0)); };
    const bool ragged = !WHOLE && (DK % V != 0 || S.dv % V != 0);
    auto mend = [&](frag &f, int d, int dim) { f = behind(f, d < dim && d > dim - V ? d - (dim - V) : 0); };
    auto load = [&](int a, int n) {
        const unsigned last = n - 1;
        const window kw = window_of(K + (long long)a * S.k_t, last * k_t + row_k), vw = window_of(Vp + (long long)a * S.v_t, last * v_t + row_v);
#pragma unroll
        for (int i = 0; i < NK; ++i) sk[i] = piece(kw, ko + i * RK * k_t);
#pragma unroll
        for (int i = 0; i < NV; ++i) sv[i] = piece(vw, vo + i * RV * v_t);
        if constexpr (!STATE_ONLY) {
            const window qw = window_of(Q + (long long)a * S.q_t, last * q_t + row_k);
#pragma unroll
            for (int i = 0; i < NK; ++i) sq[i] = piece(qw, qo + i * RK * q_t);
        }
    };
    // The starts of 64 tokens are one load and one mask; chunks do not cross their borders (`left`).
    int block = -1, asked = -1;                             // of the piece: tokens tok_a + 64 block ..; the block that `byte` is of
    unsigned long long flags = 0;
    uint8_t byte = 0;
    auto ask = [&](int k) {
        asked = k;
        const int t = tok_a + 64 * k + lane;
        byte = k >= 0 && t < tok_e ? St[(long long)t * A.a.starts_t] : 0;
    };
    auto starts_of = [&](int a, int n) -> unsigned {
        const int k = (a - tok_a) >> 6;
        if (k != block) {
            if (asked != k) ask(k);
            flags = __ballot(byte != 0);
            block = k;
            ask(rev ? k - 1 : k + 1);                       // in flight until its chunks come
        }
        return (unsigned)(flags >> ((a - tok_a) & 63)) & ((2u << (n - 1)) - 1u);
    };

    auto put = [&](window ow, frag f, unsigned off, int d) {     // elements d .. of the row at `off`; rows behind the window's end are not there
        if (!ragged || d + V <= S.dv) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, f), ow, WHOLE || d < S.dv ? off + d * (unsigned)sizeof(T) : OUTSIDE, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (d + e < S.dv) {
                    const T x = f[e];
                    const unsigned at = off + (d + e) * (unsigned)sizeof(T);
                    if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, x), ow, at, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), ow, at, 0, 0);
                }
        }
    };

    bool any_start = false;
    int pos = rev ? tok_e : tok_a, most = C;
    // (up to the next multiple of C: the first chunk of a reverse scan is the short one, and so is what follows tokens taken singly)
    auto left = [&]() {
        const int in = (pos - tok_a) & (C - 1), room = rev ? (in ? in : C) : C - in, l = rev ? pos - tok_a : tok_e - pos;
        const int n = room < most ? room : most;
        return l < n ? l : n;
    };
    // A turn of the loop writes the chunk that has been loaded to LDS, asks for the next, and computes the first.
    if (St && left() > 0) ask(rev ? (tok_e - 1 - tok_a) >> 6 : 0);
    int a = 0, n = 0;                                       // the chunk in hand: [a, a + n); none in the first turn
    for (;;) {
        const bool have = n > 0;
        float z = 0.f;
        if (have) {
            if (ragged) {
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    mend(sk[i], dk0, DK);
                    if constexpr (!STATE_ONLY) mend(sq[i], dk0, DK);
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) mend(sv[i], dvp, S.dv);
            }
        // A value that is not finite would reach other tokens through a weight of zero (0 x NaN).  Such a chunk is taken token by
        // token instead, where no token shares a product with another.  The check sums K and V on the matrix cores.
        if constexpr (TT == 2) {
            f4 z0 = {0.f, 0.f, 0.f, 0.f}, z1 = z0;
            frag one;
#pragma unroll
            for (int e = 0; e < V; ++e) one[e] = (T)1.f;
#pragma unroll
            for (int i = 0; i < NK; ++i) z0 = Y::mfma(one, sk[i], z0);
#pragma unroll
            for (int i = 0; i < NV; ++i) z1 = Y::mfma(one, sv[i], z1);
            z = z0[0] * 0.f + z1[0] * 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int i = 0; i < NK; ++i) z = __builtin_fmaf((float)sk[i][e], 0.f, z);
#pragma unroll
                for (int i = 0; i < NV; ++i) z = __builtin_fmaf((float)sv[i][e], 0.f, z);
            }
        }
        wave_sync();                                     // the chunk before has been read
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            *(frag *)(ldsK + Y::template at<DKP>(i * RK + rk, pk)) = sk[i];
            if constexpr (!STATE_ONLY) *(frag *)(ldsQ + Y::template at_rows<DKP>(i * RK + rk, pk)) = sq[i];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) *(frag *)(ldsV + Y::template at<DVS>(i * RV + rv, pv)) = sv[i];
        wave_sync();
        }
        const int pos0 = pos;
        pos += rev ? -n : n;
        most = have ? C : most;
        const int n2 = __builtin_amdgcn_readfirstlane(left()), a2 = __builtin_amdgcn_readfirstlane(rev ? pos - n2 : pos);
        if (n2 > 0) load(a2, n2);
        if (!have) {
            if (n2 <= 0) break;
            a = a2;
            n = n2;
            continue;
        }
        by_length(n);
        const unsigned mask = St ? starts_of(a, n) : 0u;
        // (starts in the chunk: x and y are of one episode if none lies behind the earlier and up to the later)
        const int start0 = mask ? __builtin_ctz(mask) : 32, start1 = mask ? 31 - __builtin_clz(mask) : 0;      // the first and the last of them
        float w[V], reach[NT];                              // wy and rx within the episodes
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = wy[e];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) reach[nt] = rx[nt];
        if (mask) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (rev ? V * g + e >= start0 : V * g + e < start1) w[e] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                if (rev ? 16 * nt + m < start1 : 16 * nt + m >= start0) reach[nt] = 0.f;
        }
        frag p[NT];
        if constexpr (!STATE_ONLY) {
            f4 at[NT][TT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < TT; ++t) at[nt][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                frag q[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) q[nt] = *(const frag *)(ldsQ + Y::template at_rows<DKP>(16 * nt + m, KP * ks + g));
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const frag k = *(const frag *)(ldsK + Y::template at<DKP>(Y::tile_row(t, m), KP * ks + g));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) at[nt][t] = Y::mfma(k, q[nt], at[nt][t]);
                }
            }
            if constexpr (AGAIN) within(here(lane) >> 4, here(lane) & 15);
            if (mask) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    // the lane's column x sees the tokens from <= y < to
                    const int x = 16 * nt + (here(lane) & 15);
                    const unsigned upto = (2u << x) - 1u, before = mask & upto, after = mask & ~upto;
                    const int from = (before && !rev ? 31 - __builtin_clz(before) : 0) - V * g, to = (after && rev ? __builtin_ctz(after) : 32) - V * g;
#pragma unroll
                    for (int t = 0; t < TT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) at[nt][t][r] = mul_or_zero(at[nt][t][r], 4 * t + r >= from && 4 * t + r < to ? dw[nt][t][r] : 0.f);
                }
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int t = 0; t < TT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) at[nt][t][r] = mul_or_zero(at[nt][t][r], dw[nt][t][r]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) p[nt] = Y::operand(at[nt]);
        }
        phase();
        frag vf[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) vf[j] = Y::template column<DVS>(ldsV, j, m, g);
        f4 o[VS][NT][TT];
        if constexpr (!STATE_ONLY) {
            // P and S as operands are rounded to the inputs' type: 2^-8 of each term at most with bf16, as much as the output's own rounding;
            // the sums, and the state that goes on, are fp32.  Outputs are off by 0.0023 of their norm then, by 0.0017 with each in two summands
            // (their own rounding).  That would cost 2 % where the card is full (128 x 2048 x 16 heads of 64: 484 us, 493), 6-9 % on windows and
            // pieces (96 x 157 x 4: 15.6, 17.1; 16384 x 8 heads of 128: 98, 106), 11-14 % where registers are short (training, 64 x 512 x 16
            // heads of 64: 227, 252; 64 x 1024 x 16 heads of 128: 301, 343).
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) o[j / TT][nt][j % TT] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                frag q[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) q[nt] = *(const frag *)(ldsQ + Y::template at_rows<DKP>(16 * nt + m, KP * ks + g));
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    f4 rows[TT];
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) rows[tt] = s[ks * TT + tt][j];
                    const frag sf = Y::operand(rows);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[j / TT][nt][j % TT] = Y::mfma(sf, q[nt], o[j / TT][nt][j % TT]);
                }
            }
        }
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    f4 &t = o[j / TT][nt][j % TT];
#pragma unroll
                    for (int r = 0; r < 4; ++r) t[r] = mul_or_zero(t[r], reach[nt]);
                    t = Y::mfma(vf[j], p[nt], t);
                }
        }
        if (__any(z != 0.f || z != z)) {
            if (n > 1) {
                pos = pos0;
                most = 1;
                n = 0;                                      // (the next turn only loads)
                continue;
            }
            // The token is alone.  What a weight of zero keeps from the state -- in a reverse scan an episode that starts with the token, or a
            // decay that remembers nothing -- is taken out of both factors of the product.
            if ((rev && mask) || S.a_write * (rev ? gn : 1.f) == 0.f) {
                frag none;
#pragma unroll
                for (int e = 0; e < V; ++e) none[e] = (T)0.f;
                wave_sync();
#pragma unroll
                for (int i = 0; i < NK; ++i) *(frag *)(ldsK + Y::template at<DKP>(i * RK + rk, pk)) = none;
                wave_sync();
#pragma unroll
                for (int j = 0; j < NJ; ++j) vf[j] = none;
            }
        }
        if constexpr (!STATE_ONLY) {
            const window ow = window_of(O + (long long)a * S.o_t, (unsigned)(n - 1) * o_t + row_v);
            if constexpr (PV <= 4 && NT == 1) {
                put(ow, Y::operand(o[0][0]), m * o_t, dv0 + g * V);
            } else {                                        // through LDS, so that neighbouring lanes store neighbouring pieces of a row
                wave_sync();
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int jg = 0; jg < VS; ++jg) *(frag *)(ldsQ + Y::template at_rows<DVS>(16 * nt + m, KP * jg + g)) = Y::operand(o[jg][nt]);
                wave_sync();
#pragma unroll
                for (int i = 0; i < NV; ++i) put(ow, *(const frag *)(ldsQ + Y::template at_rows<DVS>(i * RV + rv, pv)), (unsigned)(i * RV + rv) * o_t, dvp);
            }
        }
        // ---- the state behind the chunk
        phase();
        const bool fresh = mask != 0;
        any_start = any_start || fresh;
        const float gs = fresh ? 0.f : gn;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][j][r] = mul_or_zero(s[i][j][r], gs);
        if constexpr (NI <= 4) {                            // (K's columns: held, or with heads of 128 read again for each of V's)
            frag kt[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) kt[i] = Y::template column<DKP>(ldsK, i, m, g);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                frag part[PARTS];
                Y::template weighted<PARTS>(vf[j], w, part);
#pragma unroll
                for (int pp = 0; pp < PARTS; ++pp)
#pragma unroll
                    for (int i = 0; i < NI; ++i) s[i][j] = Y::mfma(kt[i], part[pp], s[i][j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                frag part[PARTS];
                Y::template weighted<PARTS>(vf[j], w, part);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const frag kt = Y::template column<DKP>(ldsK, i, m, g);
#pragma unroll
                    for (int pp = 0; pp < PARTS; ++pp) s[i][j] = Y::mfma(kt, part[pp], s[i][j]);
                }
                phase();
            }
        }
        if (n2 <= 0) break;
        a = a2;
        n = n2;
    }

    if constexpr (STATE_ONLY) {
        float *ws = A.a.workspace + ((long long)grp * A.n_sib + sib) * A.per_sib + lane * 4;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) *(f4 *)(ws + (i * NJ + j) * 256) = s[i][j];
        if (lane == 0 && strip == 0)
            A.carry[((long long)sc * A.a.B * A.a.H + bh) * nseg + seg] = any_start ? 0.f : power(lg, tok_e - tok_a);
    } else {
        // rows at and behind the length
        const frag zero = __builtin_bit_cast(frag, u4{0u, 0u, 0u, 0u});
        for (int t = tok_e; t < seg_e; t += RV) {
            const int rows = seg_e - t < RV ? seg_e - t : RV;
            put(window_of(O + (long long)t * S.o_t, (unsigned)(rows - 1) * o_t + row_v), zero, rv * o_t, dvp);
        }
        if ((rev ? seg == 0 : seg == nseg - 1) && S.s_out) {
            const gbytes_out p = shared_base_out(S.s_out + b * S.s_b + h * S.s_h);
            state_elements([&](int i, int j, int r, bool is, unsigned at) {
                if (is) *(__attribute__((address_space(1))) float *)(p + at) = s[i][j][r];
            });
        }
    }
}

// The states that come into the pieces, from what each piece adds: s_(i+1) = carry_i s_i + u_i, written over u_i as s_i.  A lane takes four
// elements through all pieces.  Bound: the states, read and written once (64 pieces of 8 heads of 128: 67 MB, 18 us, 3.8 TB/s; 16 or 32
// loads in flight instead of 8 take the same).
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
    auto place = [&](int n) { return (f4 *)(ws + (((long long)bh * nseg + (rev ? nseg - 1 - n : n)) * A.n_sib + sib) * A.per_sib); };
    for (int n0 = 0; n0 < nseg; n0 += 8) {                 // eight pieces' loads are in flight together
        f4 u[8];
        float c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int n = n0 + k < nseg ? n0 + k : nseg - 1;
            u[k] = *place(n);
            c[k] = carry[rev ? nseg - 1 - n : n];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (n0 + k >= nseg) break;
            *place(n0 + k) = s;
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = mul_or_zero(s[r], c[k]) + u[k][r];
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
int padded(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

// Strips are 64 value columns (32 where dk needs 128: the state has to fit the registers) if that makes a wave for every SIMD, and else
// the narrowest that fill a tile: each wave then has less to do for a chunk, and K, Q and their products are repeated.  Measured: 64
// windows of 160 x 4 heads of 64, fp32, forward 35 us wide (256 waves), 20 us narrow (1024 waves).
struct Plan { int dkp, dvs, n_sib, sib0[PVDER_SEQ_MAX_SCANS + 1]; };

bool owns(const pvder_seq_scan &s) { return !s.kept && s.transpose_of == 0; }

bool valid(const pvder_seq_attn *a) {
    if (!a || a->n_scans < 1 || a->n_scans > PVDER_SEQ_MAX_SCANS || a->B < 0 || a->T < 0 || a->T > PVDER_SEQ_MAX_TOKENS || a->H < 1) return false;
    if (a->dtype != PVDER_SEQ_F32 && a->dtype != PVDER_SEQ_BF16) return false;
    const int least = a->dtype == PVDER_SEQ_BF16 ? 8 : 4;  // 16 bytes: the kernels read rows in such pieces
    for (int i = 0; i < a->n_scans; ++i) {
        const pvder_seq_scan &s = a->scan[i];
        if (s.dk < least || s.dv < least || s.dk > PVDER_SEQ_MAX_HEAD || s.dv > PVDER_SEQ_MAX_HEAD) return false;
        if (s.transpose_of < 0 || s.transpose_of > i || (s.transpose_of && s.kept) || ((uintptr_t)s.kept & 15)) return false;
        if (s.transpose_of) {
            const pvder_seq_scan &of = a->scan[s.transpose_of - 1];
            if (!owns(of) || of.dk != s.dv || of.dv != s.dk) return false;
        }
    }
    return true;
}

// The scans of `a` whose dk has the padded size dkp (`own`: that make their own states, too), as an argument of their own, and which they
// are: scans of other sizes would be padded to the largest.
int of_size(const pvder_seq_attn *a, int dkp, bool own, pvder_seq_attn &sub, int *which) {
    sub = *a;
    sub.n_scans = 0;
    for (int i = 0; i < a->n_scans; ++i)
        if (padded(a->scan[i].dk) == dkp && (!own || owns(a->scan[i]))) {
            which[sub.n_scans] = i;
            sub.scan[sub.n_scans++] = a->scan[i];
        }
    return sub.n_scans;
}

Plan plan_of(const pvder_seq_attn *a, int dkp) {
    Plan P;
    int dv = 0;
    for (int i = 0; i < a->n_scans; ++i) dv = a->scan[i].dv > dv ? a->scan[i].dv : dv;
    P.dkp = dkp;
    const int widest = padded(dv) < 64 && dkp < 128 ? padded(dv) : (dkp == 128 ? 32 : 64), narrowest = a->dtype == PVDER_SEQ_BF16 ? 32 : 16;
    for (const int dvs : {widest, narrowest}) {
        P.dvs = dvs;
        P.n_sib = 0;
        for (int i = 0; i < a->n_scans; ++i) {
            P.sib0[i] = P.n_sib;
            P.n_sib += (a->scan[i].dv + dvs - 1) / dvs;
        }
        for (int i = a->n_scans; i <= PVDER_SEQ_MAX_SCANS; ++i) P.sib0[i] = P.n_sib;
        if ((long long)a->B * a->H * P.n_sib >= 1024) break;
    }
    return P;
}

// Whether four (b, h, piece) on end go to one XCD: where there are enough to go round, and rows of less than a line share theirs with the
// next head's (512 x 1024 x 8 heads of 32, bf16: 290 us one by one, 259 by fours, 256 by eights) or heads are of over 64 (64 x 1024 x 16 of
// 128: 327, 315, 315; of 100: 499, 476, 467; forward and backward, 32 x 1024 x 16 of 128: 598, 590, 586).  Else it is no gain: 128 x 2048 x 16 heads of 64 486, 491, 504; 64 windows of 160 x 4 heads of 64, fp32, 61.5, 63, 63.
bool fours(const pvder_seq_attn &a, unsigned n_groups, int dkp) {
    bool shared = dkp == 128 && a.segments == 1;
    for (int i = 0; i < a.n_scans; ++i) shared = shared || (a.scan[i].dk < a.scan[i].dv ? a.scan[i].dk : a.scan[i].dv) * (a.dtype == PVDER_SEQ_BF16 ? 2 : 4) < 128;
    return shared && n_groups >= 256;
}

long long scan_blocks(long long n_groups, unsigned together_log2, int n_sib) {
    const long long deal = 8ll << together_log2;
    return (n_groups + deal - 1) / deal * deal * n_sib;
}
long long join_items(const pvder_seq_attn &a, int n_sib, int dkp, int dvs) { return (long long)a.B * a.H * n_sib * (dkp * dvs / 4); }

// Whether the threads of each launch that a call with `rows` batch rows makes can be counted
bool countable(const pvder_seq_attn *a, int rows) {
    const long long n = (long long)rows * a->H;
    if (n > kMostThreads || n * a->segments > kMostThreads) return false;
    pvder_seq_attn all = *a, sub;
    all.B = rows;
    int which[PVDER_SEQ_MAX_SCANS];
    for (const bool first : {true, false})
        for (const int dkp : {32, 64, 128}) {
            if ((first && a->segments < 2) || !of_size(&all, dkp, first, sub, which)) continue;
            const Plan P = plan_of(&sub, dkp);
            if (scan_blocks(n * a->segments, 2, P.n_sib) > kMostThreads / 64) return false;
            if (first && join_items(sub, P.n_sib, P.dkp, P.dvs) > kMostThreads - 255) return false;
        }
    return true;
}

int64_t workspace_of(const pvder_seq_attn *a, const Plan &P) {
    const int64_t bhs = (int64_t)a->B * a->H * a->segments;
    return (bhs * P.n_sib * P.dkp * P.dvs + bhs * a->n_scans + 3) / 4 * 4;      // (whole 16 bytes: the next size's begins there)
}

int seg_len_of(const pvder_seq_attn *a) {
    const int c = 32, per = (a->T + a->segments - 1) / a->segments;
    return (per + c - 1) / c * c;
}

// The states of one scan of `a` among those that a plan lays into `at`
States states_of(const float *at, const Plan &P, int scan, int dv, bool transposed) {
    const long long strip = (long long)P.dkp * P.dvs;
    const int side = P.dvs / 16;
    return States{at + P.sib0[scan] * strip, P.n_sib * strip, side == 4 ? 2 : side - 1, (dv + P.dvs - 1) / P.dvs, P.dkp / 16, transposed};
}

// `states`: what each piece adds to the state and from that the states that come into the pieces; else the outputs
template <typename T, int DKP, int DVS, bool WHOLE> int launch(const Args &A, bool states, hipStream_t st) {
    constexpr int MOST = sizeof(T) == 2 ? 3 : 1, LEAST = sizeof(T) == 2 ? 2 : 1;
    const dim3 grid((unsigned)scan_blocks(A.n_groups, A.together_log2, A.n_sib)), block(64);
    const int bytes = tile_bytes<T>(DKP, DVS);
    if (states) {
        const long long items = join_items(A.a, A.n_sib, DKP, DVS);
        seq_scan_kernel<T, DKP, DVS, WHOLE, true, MOST><<<grid, block, bytes, st>>>(A);
        seq_join_kernel<T, DKP, DVS><<<dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st>>>(A);
    } else {
        bool state = false;
        for (int i = 0; i < A.a.n_scans; ++i) state = state || A.a.scan[i].s_out != nullptr;
        if (state) seq_scan_kernel<T, DKP, DVS, WHOLE, false, MOST><<<grid, block, bytes, st>>>(A);
        else seq_scan_kernel<T, DKP, DVS, WHOLE, false, LEAST><<<grid, block, bytes, st>>>(A);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -(int)e;
}

template <typename T, int DKP, int DVS> int fit(const Args &A, bool states, hipStream_t st) {
    bool whole = true;
    for (int i = 0; i < A.a.n_scans; ++i) whole = whole && A.a.scan[i].dk == DKP && A.a.scan[i].dv % DVS == 0;
    return whole ? launch<T, DKP, DVS, true>(A, states, st) : launch<T, DKP, DVS, false>(A, states, st);
}

template <typename T> int pick(const Args &A, const Plan &P, bool states, hipStream_t st) {
    constexpr int NARROW = sizeof(T) == 2 ? 32 : 16;
    if (P.dkp == 32)
        return P.dvs == 64 ? fit<T, 32, 64>(A, states, st) : (P.dvs == 32 ? fit<T, 32, 32>(A, states, st) : fit<T, 32, NARROW>(A, states, st));
    if (P.dkp == 64)
        return P.dvs == 64 ? fit<T, 64, 64>(A, states, st) : (P.dvs == 32 ? fit<T, 64, 32>(A, states, st) : fit<T, 64, NARROW>(A, states, st));
    return P.dvs == 32 ? fit<T, 128, 32>(A, states, st) : fit<T, 128, NARROW>(A, states, st);
}

// All launches of a call whose arguments have been checked
int run_rows(const pvder_seq_attn *a, hipStream_t st) {
    Args A = {};
    const bool pieces = a->segments > 1 && a->T > 0;
    States states[PVDER_SEQ_MAX_SCANS];
    float *work = a->workspace;
    int which[PVDER_SEQ_MAX_SCANS];
    for (const bool first : {true, false}) {               // the states of all pieces, then the outputs
        if (first && !pieces) continue;
        for (const int dkp : {32, 64, 128}) {
            if (!of_size(a, dkp, first, A.a, which)) continue;
            if (!pieces) A.a.segments = 1;
            const Plan P = plan_of(&A.a, dkp);
            A.seg_len = A.a.T ? seg_len_of(&A.a) : 32;
            A.n_sib = P.n_sib;
            for (int i = 0; i <= PVDER_SEQ_MAX_SCANS; ++i) A.sib0[i] = P.sib0[i];
            A.n_groups = (unsigned)((long long)a->B * a->H * A.a.segments);
            A.together_log2 = fours(A.a, A.n_groups, dkp) ? 2 : 0;
            A.per_sib = (long long)P.dkp * P.dvs;
            if (first) {
                A.a.workspace = work;
                A.carry = work + (long long)A.n_groups * P.n_sib * A.per_sib;
                work += workspace_of(&A.a, P);
                for (int i = 0; i < A.a.n_scans; ++i) states[which[i]] = states_of(A.a.workspace, P, i, A.a.scan[i].dv, false);
            } else if (pieces) {
                for (int i = 0; i < A.a.n_scans; ++i) {
                    const pvder_seq_scan &s = A.a.scan[i];
                    if (s.kept) {
                        pvder_seq_attn was = *a;           // the run that left them
                        was.n_scans = 1;
                        was.scan[0].dk = s.dv;
                        was.scan[0].dv = s.dk;
                        A.states[i] = states_of(s.kept, plan_of(&was, padded(s.dv)), 0, s.dk, true);
                    } else if (s.transpose_of) {
                        A.states[i] = states[s.transpose_of - 1];
                        A.states[i].transposed = true;
                    } else {
                        A.states[i] = states[which[i]];
                    }
                }
            }
            const int rc = a->dtype == PVDER_SEQ_BF16 ? pick<__bf16>(A, P, first, st) : pick<float>(A, P, first, st);
            if (rc) return rc;
        }
    }
    return 0;
}

}  // namespace

extern "C" int64_t pvder_seq_attn_plan(pvder_seq_attn *a) {
    if (!valid(a)) return kEinval;
    pvder_seq_attn sub;
    int which[PVDER_SEQ_MAX_SCANS];
    bool given = false;
    for (int i = 0; i < a->n_scans; ++i) given = given || a->scan[i].kept;
    if (given && a->segments < 2) return kEinval;
    // Pieces of T side by side cost a second reading of K and V, a state of each piece in memory and two more launches: worth it where
    // the waves leave most of the card idle and the pieces make up for it.  Measured at heads of 64, bf16, one piece against the rule's:
    // 16 waves of 2048 tokens 82 us and 22 (32 pieces), 128 waves 84 and 35 (8); 512 waves 86 and 100 (4), 1024 waves of 512 61 and 86 (2).
    // With states that are there already pieces pay up to twice as many waves: forward and backward, 768 waves of 2048 tokens in the
    // backward pass 262 us in one piece and 236 (fp32), 155 and 157 (bf16), 1152 waves of 1024 110 and 122.
    long long waves = 0;
    for (const int dkp : {32, 64, 128})
        if (of_size(a, dkp, false, sub, which)) waves += (long long)a->B * a->H * plan_of(&sub, dkp).n_sib;
    if (given) {
        if (waves > 768) a->segments = 1;
    } else {
        a->segments = 1;
        if (waves >= 1 && waves <= 384 && a->T >= 384) {
            const long long want = 2048 / waves, most = a->T / 64, n = want < most ? want : most;
            if (n >= 4) a->segments = (int32_t)n;
        }
    }
    if (a->segments == 1) return 0;
    int64_t floats = 0;
    for (const int dkp : {32, 64, 128})
        if (of_size(a, dkp, true, sub, which)) floats += workspace_of(&sub, plan_of(&sub, dkp));
    return floats;
}

extern "C" int pvder_seq_attn_run(const pvder_seq_attn *a, void *stream) {
    // (more pieces than the plan makes would have tokens past 32 bits)
    if (!valid(a) || a->segments < 1 || (a->segments > 1 && a->segments > a->T / 64) || !a->log_decay) return kEinval;
    bool work_needed = false;
    for (int i = 0; i < a->n_scans; ++i) work_needed = work_needed || (a->segments > 1 && owns(a->scan[i]));
    if (work_needed && (!a->workspace || ((uintptr_t)a->workspace & 15))) return kEinval;
    for (int i = 0; i < a->n_scans; ++i) {                  // (states go in and out also where there is no token)
        const pvder_seq_scan &s = a->scan[i];
        if ((s.s_in || s.s_out) && (s.s_k < 0 || s.s_v < 0 || s.s_k >= (1ll << 29) || s.s_v >= (1ll << 29) || s.dk * s.s_k + s.dv * s.s_v >= (1ll << 29))) return kEinval;
    }
    if (a->B > 0 && a->T > 0) {
        const int64_t most = PVDER_SEQ_MAX_TOKEN_STRIDE / (a->dtype == PVDER_SEQ_BF16 ? 2 : 4);
        for (int i = 0; i < a->n_scans; ++i) {
            const pvder_seq_scan &s = a->scan[i];
            if (!s.q || !s.k || !s.v || !s.o) return kEinval;
            // (a row's end, where the window of a chunk ends, has to lie before the next row)
            if (s.q_t < s.dk || s.k_t < s.dk || s.v_t < s.dv || s.o_t < s.dv || s.q_t > most || s.k_t > most || s.v_t > most || s.o_t > most) return kEinval;
            if (s.transpose_of) {
                const pvder_seq_scan &of = a->scan[s.transpose_of - 1];
                if (s.k != of.v || s.v != of.k || s.reverse != of.reverse || s.a_write != of.a_write) return kEinval;
            }
        }
    }
    if (a->B == 0) return 0;
    // as many batch rows at once as the threads of a launch can be counted for (few rows of few heads, where T is in pieces)
    int rows = a->B;
    while (!countable(a, rows)) {
        if (rows == 1 || (a->segments > 1 && a->T > 0)) return kEinval;
        rows -= rows / 2;
    }
    const long long es = a->dtype == PVDER_SEQ_BF16 ? 2 : 4;
    for (long long b = 0; b < a->B; b += rows) {
        pvder_seq_attn part = *a;
        part.B = (int32_t)(a->B - b < rows ? a->B - b : rows);
        for (int i = 0; i < a->n_scans; ++i) {
            pvder_seq_scan &s = part.scan[i];
            s.q = (const char *)s.q + b * s.q_b * es;
            s.k = (const char *)s.k + b * s.k_b * es;
            s.v = (const char *)s.v + b * s.v_b * es;
            s.o = (char *)s.o + b * s.o_b * es;
            if (s.s_in) s.s_in += b * s.s_b;
            if (s.s_out) s.s_out += b * s.s_b;
        }
        if (a->starts) part.starts = a->starts + b * a->starts_b;
        if (a->lengths) part.lengths = a->lengths + b;
        const int rc = run_rows(&part, (hipStream_t)stream);
        if (rc) return rc;
    }
    return 0;
}
