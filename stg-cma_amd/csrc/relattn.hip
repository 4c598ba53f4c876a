// Attention over ragged token sequences with a learned relative position bias by buckets: forward, backward (dQ, dK, dV and the
// bias table's gradient) and the single-token form over a key / value cache.  The additive term depends on the signed distance
// between key and query position alone, through a table of a few buckets per head (single distances near zero, then buckets evenly
// spaced in the logarithm up to a border behind which every distance shares the last one), so it is never formed as [n, n]:
//     x_ij = scale q_i . k_j + table[bucket(j - p_i)][h],  p_i = i + (n_k - n_q),   P = softmax(x),   O = P V.
//
// Sequence s owns query rows cu_q[s] .. cu_q[s+1] - 1 and key rows cu_k[s] .. cu_k[s+1] - 1 of packed row tensors; heads share
// key / value heads (H % Hkv == 0); key_mask and the causal rule hide keys; a query that sees no key gives a zero row, lse = -inf
// and no gradient.  Rows of masked keys and rows past a sequence's end enter LDS as zeros, so whatever they hold stays out.
//
// How the bias costs (almost) nothing: a block spreads its head's row of the table into LDS once, indexed by distance, divided by
// the scale; a tile whose distances all lie behind the last border starts the score MFMA's accumulator at ONE constant, a nearer tile
// starts it at 16 LDS words per lane (consecutive lanes read consecutive words).  Neither adds an instruction to the softmax.
//
// MFMA v_mfma_f32_32x32x16_bf16; lane l = (r = l & 31, hh = l >> 5); accumulator row (reg, hh) = (reg & 3) + 8 (reg >> 2) + 4 hh.
#include <math.h>
#include <type_traits>
#include "common.h"
#include "../../include/stgcma.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int PAD = 96;               // a 64 x 32 tile that touches distance +-(far - 1) reaches at most 94 beyond it

constexpr int TAIL_LSE = 2;           // zero_tail: the forward clears the rows of lse alone, the backward nothing
struct RP {
    const bf16_t* Q; int64_t ldq;
    const bf16_t* K; int64_t ldk;
    const bf16_t* V; int64_t ldv;
    bf16_t* O; int64_t ldo;
    float* lse;                       // [H, Tq], natural logarithm
    const int32_t* cu_q; const int32_t* cu_k;
    const uint8_t* kmask;
    int64_t Tq, Tk;
    int S, H, Hkv, causal, zero_tail;
    const float* table; const int32_t* plan;
    int NB, far;
    float scale, scale2, inv_scale;
    const bf16_t* dO; int64_t lddo;
    bf16_t* dQ; int64_t lddq;
    bf16_t* dK; int64_t lddk;
    bf16_t* dV; int64_t lddv;
    float* delta;                     // [H, Tq]
    float* fix;                       // [H, Tq]: what the score of a row far out (BIG_LSE) needs beside lse, in raw units; other rows' entries are not set
    uint32_t* seen; int qtiles;       // [S, H, qtiles, 4]: what a wave of the dQ kernel saw (FAR_OUT, LONE); that kernel's `tiles`
    float* part;                      // partial table gradients: [S * tiles, H, 2] behind the borders / [S * tiles, H, NB] of the band; or NULL
    int tiles;                        // blocks per (sequence, head)
    int hsplit;                       // dK / dV: blocks that share the heads of one key / value head
    float* pk;                        // their parts [hsplit][dK, dV][Tk, Hkv D], when there are several
};

// Which (tile, head, sequence) a block of the one-dimensional grid serves; the blocks that clear the rows behind the last sequence (s == S) come
// last.  Without the causal rule tiles run fastest: neighbouring blocks share their keys in L2.  With it heads run fastest, then sequences, and the
// heaviest tiles come first, so the long walks do not start last; the sequence is rotated by the tile, since consecutive blocks go to the
// eight XCDs in turn and a fixed order would hand the long sequences to the same ones (measured with sequences fastest: 1.7 times slower).
struct Who { int tile, h, s; };
__device__ __forceinline__ Who who(const RP& a, int heads) {
    const int id = blockIdx.x;
    Who w;
    if (a.causal) {
        const int u = id / heads;
        w.h = id % heads;
        w.tile = a.S > 0 ? u / a.S : a.tiles;
        if (w.tile < a.tiles) w.s = (u % a.S + w.tile) % a.S;
        else { w.tile = u - a.tiles * a.S; w.s = a.S; }
    } else {
        w.tile = id % a.tiles;
        w.h = id / a.tiles % heads;
        w.s = id / a.tiles / heads;
    }
    return w;
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));
#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16((a), (b), (c), 0, 0, 0)
#define ACC_ROW(reg, hh) (((reg) & 3) + 8 * ((reg) >> 2) + 4 * (hh))

__device__ __forceinline__ bf16x8_t ld_frag(const bf16_t* p) { return *reinterpret_cast<const bf16x8_t*>(p); }
__device__ __forceinline__ f32x16_t splat16(float v) {
    f32x16_t z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = v;
    return z;
}
// maxima that hand a NaN on (v_maximum3_f32: no canonicalisation of the MFMA results in front of it)
__device__ __forceinline__ float fmax2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float fmax3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
// the other half-wave's value meets the lane's own (lanes r and r + 32 hold the two halves of a query's or key's accumulator rows)
__device__ __forceinline__ void both_halves(float v, float& lo, float& hi) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lo = __uint_as_float(w[0]);
    hi = __uint_as_float(w[1]);
}
__device__ __forceinline__ float half_sum(float v) { float a, b; both_halves(v, a, b); return a + b; }
__device__ __forceinline__ float half_max(float v) { float a, b; both_halves(v, a, b); return fmax2(a, b); }
// Operands loaded in front of a loop have arrived before it is entered.  (Without a use here the wait-count bookkeeping takes them as possibly in flight on
// some path into the loop, and every trip's first products then wait for the NEXT tile's loads, which were issued behind them.)
template <int N> __device__ __forceinline__ void arrived(bf16x8_t (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}
__device__ __forceinline__ bf16x8_t zero_frag() { const u32x4_t z = {0u, 0u, 0u, 0u}; return __builtin_bit_cast(bf16x8_t, z); }
__device__ __forceinline__ bf16x8_t pack8(const float* x) {
    const u32x4_t w = {pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7])};
    return __builtin_bit_cast(bf16x8_t, w);
}
// transposed fragment of a [rows][DP] tile: A[i = d][k slot j] = tile[16 s2 + 4 hh + (j & 3) + 8 (j >> 2)][32 dt + d]
template <int DP>
__device__ __forceinline__ bf16x8_t tr_frag(const bf16_t* s, int dt, int s2, int hh, int d) {
    const int gi = d & 15, c = d >> 4;
    const bf16_t* p = s + (16 * s2 + 4 * hh + (gi >> 2)) * DP + 32 * dt + 16 * c + 4 * (gi & 3);
    const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p);
    const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)(p + 8 * DP));
    bf16x8_t f;
    f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
    f[4] = hi[0]; f[5] = hi[1]; f[6] = hi[2]; f[7] = hi[3];
    return f;
}
template <int DP>
__device__ __forceinline__ bf16x8_t nat_frag(const bf16_t* s, int r, int hh, int ks) {
    return *reinterpret_cast<const bf16x8_t*>(s + r * DP + 16 * ks + 8 * hh);
}

struct Seq { int q0, nq, k0, nk; };
// The offsets come from device memory: whatever they hold, the rows stay inside the tensors (sequence 0 starts at row 0).
__device__ __forceinline__ Seq seq_of(const RP& a, int s) {
    const int tq = (int)a.Tq, tk = (int)a.Tk;
    auto clampi = [](int v, int hi) { return v < 0 ? 0 : (v > hi ? hi : v); };
    Seq z;
    z.q0 = s == 0 ? 0 : clampi(a.cu_q[s], tq);
    z.nq = clampi(a.cu_q[s + 1], tq) - z.q0;
    z.k0 = s == 0 ? 0 : clampi(a.cu_k[s], tk);
    z.nk = clampi(a.cu_k[s + 1], tk) - z.k0;
    z.nq = z.nq < 0 ? 0 : z.nq;
    z.nk = z.nk < 0 ? 0 : z.nk;
    return z;
}

// A table entry in units of the raw score.  Entries at or below -1e30 (the type's lowest value, a common mask) hide their bucket like -inf: as
// scores they would swallow q.k in fp32.  Other finite entries are held within +-1e8, where a row maximum's own rounding (at most 8 in the
// exponent, common to the row) leaves every power of two in range and cancels in the normalisation: by the row's sum in the forward, by the sum of the
// recomputed probabilities in the backward (BIG_LSE).
__device__ __forceinline__ float raw_bias(float t, float inv_scale) {
    if (t <= -1e30f) return -INFINITY;
    if (t < -1e8f) t = -1e8f;
    if (t > 1e8f && t < INFINITY) t = 1e8f;
    return t * inv_scale;
}
// bv[i] = bias of distance i - (far + PAD); distances past the border hold its value.  Under the causal rule no tile reaches more than 94 keys behind a
// query (heads of 128, distances up to 2000: two blocks to a compute unit instead of one: 4 x 4096 x 16 heads 598 -> 400 us)
__host__ __device__ __forceinline__ int bias_len(int far, bool causal) { return far + PAD + (causal ? PAD : far + PAD) + 1; }
__device__ __forceinline__ void fill_bias(const RP& a, int h, float* bv, int tid, int nthr) {
    const int len = bias_len(a.far, a.causal);
    for (int i = tid; i < len; i += nthr) {
        int d = i - (a.far + PAD);
        d = d < -a.far ? -a.far : (d > a.far ? a.far : d);
        int b = a.plan[d + a.far];
        b = b < 0 ? 0 : (b < a.NB ? b : a.NB - 1);
        bv[i] = raw_bias(a.table[(int64_t)b * a.H + h], a.inv_scale);
    }
}

// Staging of two [64][D] tiles (K and V, or Q and dO) by NTHR threads in 16-byte pieces through registers.  A thread's pieces are rows
// of one column piece: one 32-bit byte offset per tensor and scalar bases, so a full tile costs no address arithmetic.  (D = 96: 256 threads are no
// whole number of rows; an offset per piece.)
template <int N> using U4Arr = u32x4_t[N];
template <int D, int NTHR> struct StageC {
    static constexpr int ROWP = D / 8;                       // pieces per row
    static constexpr int HALF = 64 * ROWP / NTHR;            // pieces of one tensor per thread
    static constexpr int PER = 2 * HALF;
    static constexpr int STEP = NTHR % ROWP == 0 ? NTHR / ROWP : 0;     // rows between a thread's pieces, 0: not one number
    static constexpr int NOFF = STEP ? 1 : HALF;
    static constexpr int DP = D + 8;                         // padded pitch: conflict-free for row-wise reads; transposed ones conflict two-way at 64, four-way at 128
                                                             // (10 % and 25 % as many conflict cycles as busy ones in the forward)
    static constexpr int TILE = 64 * DP;
    static_assert(64 * ROWP % NTHR == 0, "every thread moves the same number of pieces");
};
template <int D, int NTHR> __device__ __forceinline__ int stage_row(int tid, int i) { return (tid + NTHR * i) / StageC<D, NTHR>::ROWP; }
template <int D, int NTHR> __device__ __forceinline__ int stage_col(int tid, int i) { return 8 * ((tid + NTHR * i) % StageC<D, NTHR>::ROWP); }
template <int D, int NTHR>
__device__ __forceinline__ void stage_one(u32x4_t* v, int tid, const bf16_t* t, int64_t ld, const uint32_t* off, int row0, int n) {
    using C = StageC<D, NTHR>;
    if (row0 + 64 <= n) {
        const char* base = reinterpret_cast<const char*>(t + (int64_t)row0 * ld);
#pragma unroll
        for (int i = 0; i < C::HALF; ++i) v[i] = *reinterpret_cast<const u32x4_t*>(base + (C::STEP ? (int64_t)i * C::STEP * ld * 2 : 0) + off[C::STEP ? 0 : i]);
    } else {                                                 // the last tile: rows past the end read the last row (and are zeroed on the way into LDS)
#pragma unroll
        for (int i = 0; i < C::HALF; ++i) {
            int row = row0 + stage_row<D, NTHR>(tid, i);
            row = row < n ? row : n - 1;
            v[i] = *reinterpret_cast<const u32x4_t*>(t + (int64_t)row * ld + stage_col<D, NTHR>(tid, i));
        }
    }
}
template <int D, int NTHR> struct Stage {
    using C = StageC<D, NTHR>;
    uint32_t off0[C::NOFF], off1[C::NOFF];
    __device__ __forceinline__ void plan(int tid, int64_t ld0, int64_t ld1) {
#pragma unroll
        for (int i = 0; i < C::NOFF; ++i) {
            off0[i] = 2 * ((uint32_t)stage_row<D, NTHR>(tid, i) * (uint32_t)ld0 + stage_col<D, NTHR>(tid, i));
            off1[i] = 2 * ((uint32_t)stage_row<D, NTHR>(tid, i) * (uint32_t)ld1 + stage_col<D, NTHR>(tid, i));
        }
    }
    // one of the two tensors into HALF registers
    __device__ __forceinline__ void fetch1(U4Arr<C::HALF>& v, int tid, const bf16_t* t, int64_t ld, int which, int row0, int n) const {
        stage_one<D, NTHR>(v, tid, t, ld, which ? off1 : off0, row0, n);
    }
    __device__ __forceinline__ void fetch(U4Arr<C::PER>& v, int tid, const bf16_t* t0, int64_t ld0, const bf16_t* t1, int64_t ld1, int row0, int n) const {
        stage_one<D, NTHR>(v, tid, t0, ld0, off0, row0, n);
        stage_one<D, NTHR>(v + C::HALF, tid, t1, ld1, off1, row0, n);
    }
};
// `valid`: bit r set = row r of the tile takes part; other rows are written as zeros
template <int D, int NTHR>
__device__ __forceinline__ void commit_one(bf16_t* s, u32x4_t* v, int tid, uint64_t valid) {
    using C = StageC<D, NTHR>;
    if (valid != ~0ull) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < C::HALF; ++i)
            if (!((valid >> stage_row<D, NTHR>(tid, i)) & 1)) v[i] = (u32x4_t){0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < C::HALF; ++i) *reinterpret_cast<u32x4_t*>(s + stage_row<D, NTHR>(tid, i) * C::DP + stage_col<D, NTHR>(tid, i)) = v[i];
}
template <int D, int NTHR>
__device__ __forceinline__ void stage_commit(bf16_t* s, U4Arr<StageC<D, NTHR>::PER>& v, int tid, uint64_t valid) {
    commit_one<D, NTHR>(s, v, tid, valid);
    commit_one<D, NTHR>(s + StageC<D, NTHR>::TILE, v + StageC<D, NTHR>::HALF, tid, valid);
}
// The 64 keys kb .. kb + 63 of a sequence that exist and are not masked: key_load asks for the lane's mask byte (nothing looks at it yet: the load stays
// in flight), key_bits makes the wave-uniform bits of them.
__device__ __forceinline__ int key_load(const RP& a, const Seq& z, int kb, int lane) {
    if (a.kmask == nullptr) return 1;
    const int key = kb + lane < z.nk ? kb + lane : z.nk - 1;
    return a.kmask[(int64_t)z.k0 + key];
}
__device__ __forceinline__ uint64_t key_bits(const RP& a, const Seq& z, int byte, int kb, int lane) {
    const uint64_t b = __builtin_amdgcn_ballot_w64((byte != 0 || a.kmask == nullptr) && kb + lane < z.nk);
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
}
// A sequence in which at most one key is visible: a row's only probability is one and dS is zero, not what its terms' roundings leave of them.  Asked where the
// first 64 keys show at most one (`few`); ends at the second visible key, four loads in flight (a mask may hide a long beginning).
__device__ __forceinline__ bool few(uint64_t bits) { return (bits & (bits - 1)) == 0; }
__device__ __forceinline__ bool lone_key(const RP& a, const Seq& z, int lane) {
    if (z.nk <= 1) return true;
    if (a.kmask == nullptr) return false;
    bool one = false;
#pragma unroll 1
    for (int64_t k0 = 0; k0 < z.nk; k0 += 256) {
        const int kb = (int)k0;
        int byte[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) byte[i] = key_load(a, z, kb + 64 * i, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t b = key_bits(a, z, byte[i], kb + 64 * i, lane);
            if (!few(b) || (b != 0 && one)) return false;
            one = one || b != 0;
        }
    }
    return true;
}
// start of a score accumulator: bias of rows kb + ACC_ROW(., hh) against the lane's query position (idx = bv index of row 0, hh included)
__device__ __forceinline__ f32x16_t bias16(const float* bv, int idx) {
    f32x16_t c;
#pragma unroll
    for (int reg = 0; reg < 16; ++reg) c[reg] = bv[idx + (reg & 3) + 8 * (reg >> 2)];
    return c;
}

// rows behind the last sequence: zeros (and lse = -inf), when the caller owns no content there
__device__ __forceinline__ void zero_rows(bf16_t* t, int64_t ld, int64_t from, int64_t to, int col0, int D, int step, int off) {
    const int per = D / 8;
    for (int64_t i = off; i < (to - from) * per; i += step) {
        const int64_t row = from + i / per;
        *reinterpret_cast<u32x4_t*>(t + row * ld + col0 + 8 * (int)(i % per)) = (u32x4_t){0u, 0u, 0u, 0u};
    }
}
__device__ __forceinline__ int64_t tail_start(const int32_t* cu, int S, int64_t T) {
    const int64_t e = S > 0 ? cu[S] : 0;
    return e < 0 ? 0 : (e > T ? T : e);
}

// ------------------------------------------------------------------------------------------------ forward
// A block = one (sequence, head) and 32 NW queries, 32 per wave; K / V in 64-key tiles, double-buffered in LDS, one barrier per tile.
// Scores are computed transposed (rows = keys, lane = query): the softmax statistics are lane-local and P feeds the second MFMA from
// registers.
// Bound by issue: exponentials and their packing (a dozen VALU slots per score and four lanes) beside the products, 38 % of the cycles in
// the matrix units at D = 64, 33 % at D = 128.  1.35 ms = 0.81 PFLOP/s (one sequence of 16384, 16 heads of 64), 0.30 ms = 0.70 PFLOP/s
// (causal, 1311 .. 4097 x 32 / 8 heads of 128), 0.105 ms = 0.54 (985 .. 1970, 8 heads of 96).  Tiles of 64 queries and two waves: 1.8 times slower at every
// length (K and V staged twice as often by half the threads).
template <int D, int NW>
__global__ void __launch_bounds__(NW * 64, D <= 64 ? 3 : 2) relattn_fwd_kernel(RP a) {
    constexpr int KS = D / 16, DT = D / 32, DP = D + 8, NTHR = NW * 64;
    using SC = StageC<D, NTHR>;
    extern __shared__ __attribute__((aligned(16))) bf16_t smem[];       // two buffers x {K, V} x [64][DP], then the bias by distance
    float* bv = reinterpret_cast<float*>(smem + 4 * SC::TILE);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // (wave-uniform for the compiler too)
    const int r = lane & 31, hh = lane >> 5;
    const Who w = who(a, a.H);
    const int h = w.h, hk = h / (a.H / a.Hkv);
    if (w.s == a.S) {                                       // the slice that clears the rows behind the last sequence
        const int64_t from = tail_start(a.cu_q, a.S, a.Tq);
        const int step = a.tiles * NTHR, off = w.tile * NTHR + tid;
        if (a.zero_tail != TAIL_LSE) zero_rows(a.O, a.ldo, from, a.Tq, h * D, D, step, off);
        if (a.lse) for (int64_t i = from + off; i < a.Tq; i += step) a.lse[(int64_t)h * a.Tq + i] = -INFINITY;
        return;
    }
    const Seq z = seq_of(a, w.s);
    const int shift = z.nk - z.nq;
    Stage<D, NTHR> sg;
    sg.plan(tid, a.ldk, a.ldv);
    bool filled = false;
    for (int64_t tile = w.tile; tile * 32 * NW < z.nq; tile += a.tiles) {
        // heavy tiles first under the causal rule
        const int nt = (z.nq + 32 * NW - 1) / (32 * NW);
        const int qt = a.causal ? nt - 1 - (int)tile : (int)tile;
        const int qw = 32 * (qt * NW + wave);                           // first query of the wave
        const bool live = qw < z.nq;
        const int q = qw + r;
        const int64_t qrow = (int64_t)z.q0 + (q < z.nq ? q : z.nq - 1);
        const int plo = qw + shift, phi = plo + 31, pos = plo + r;      // positions of the wave's queries
        bf16x8_t qf[KS];
        {
            const bf16_t* qp = a.Q + qrow * a.ldq + h * D + 8 * hh;
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = ld_frag(qp + 16 * s);
        }
        f32x16_t o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = splat16(0.f);
        float m = -INFINITY, l = 0.f;

        int kend = z.nk;                                                // keys any query of the block may see
        if (a.causal) {
            const int last = qt * 32 * NW + 32 * NW - 1 + shift + 1;
            kend = kend < last ? kend : (last < 0 ? 0 : last);
        }
        const int np = (kend + 63) >> 6;
        const bf16_t* Kb = a.K + (int64_t)z.k0 * a.ldk + hk * D;
        const bf16_t* Vb = a.V + (int64_t)z.k0 * a.ldv + hk * D;
        u32x4_t sv[SC::PER];
        uint64_t bits = 0;
        int mk = 0;
        if (np > 0) {
            mk = key_load(a, z, 0, lane);
            sg.fetch(sv, tid, Kb, a.ldk, Vb, a.ldv, 0, z.nk);
        }
        if (!filled) { fill_bias(a, h, bv, tid, NTHR); filled = true; }
        if (np > 0) {
            bits = key_bits(a, z, mk, 0, lane);
            stage_commit<D, NTHR>(smem, sv, tid, bits);
        }
        __syncthreads();
        float cleft = bv[0], cright = bv[bias_len(a.far, a.causal) - 1];
        arrived(qf);
        asm volatile("" : "+v"(cleft), "+v"(cright));
        for (int kp = 0; kp < np; ++kp) {
            const bf16_t* sK = smem + (kp & 1) * 2 * SC::TILE;
            const bf16_t* sV = sK + SC::TILE;
            const int kb = 64 * kp;
            if (kp + 1 < np) {
                mk = key_load(a, z, kb + 64, lane);
                sg.fetch(sv, tid, Kb, a.ldk, Vb, a.ldv, kb + 64, z.nk);
            }
            if (live && bits != 0 && !(a.causal && kb > phi)) {
                // St[key][q] of keys kb .. + 31 / + 32 .. + 63.  Behind a border the bias is one number: it joins the exponent's constant and
                // the MFMA starts at zero; nearer, the accumulator starts at the bias.
                f32x16_t sA, sB;
                __builtin_amdgcn_s_setprio(1);                          // products before the other waves' exponentials: 1 .. 4 % (in dQ: nothing)
                float far = 0.f;
                const bool left = kb + 63 - plo <= -a.far;
                if (left || kb - phi >= a.far) {
                    far = left ? cleft : cright;
                    sA = MFMA32(nat_frag<DP>(sK, r, hh, 0), qf[0], splat16(0.f));
                    sB = MFMA32(nat_frag<DP>(sK + 32 * DP, r, hh, 0), qf[0], splat16(0.f));
                } else {
                    const int idx = kb + 4 * hh - pos + a.far + PAD;
                    sA = MFMA32(nat_frag<DP>(sK, r, hh, 0), qf[0], bias16(bv, idx));
                    sB = MFMA32(nat_frag<DP>(sK + 32 * DP, r, hh, 0), qf[0], bias16(bv, idx + 32));
                }
#pragma unroll
                for (int s = 1; s < KS; ++s) {
                    sA = MFMA32(nat_frag<DP>(sK, r, hh, s), qf[s], sA);
                    sB = MFMA32(nat_frag<DP>(sK + 32 * DP, r, hh, s), qf[s], sB);
                }
                __builtin_amdgcn_s_setprio(0);
                if (bits != ~0ull || (a.causal && kb + 63 > plo)) {
                    uint64_t vis = bits;                                // keys this lane's query may see
                    if (a.causal) {
                        const int c = pos - kb;                         // last visible key of the tile
                        vis = c < 0 ? 0 : (c >= 63 ? vis : vis & ((2ull << c) - 1));
                    }
                    vis >>= 4 * hh;
#pragma unroll
                    for (int reg = 0; reg < 16; ++reg) {
                        sA[reg] = (vis >> ACC_ROW(reg, 0)) & 1 ? sA[reg] : -INFINITY;
                        sB[reg] = (vis >> (32 + ACC_ROW(reg, 0))) & 1 ? sB[reg] : -INFINITY;
                    }
                }
                float mr = fmax3(sA[0], sB[0], sA[1]);                  // the maximum on the raw scores (scale > 0)
                mr = fmax3(mr, sB[1], sB[2]);
#pragma unroll
                for (int reg = 2; reg < 15; ++reg) mr = fmax3(mr, sA[reg], sB[reg + 1]);
                mr = fmax2(mr, sA[15]);
                mr = half_max(mr) + far;
                // The reference follows the maximum only once some query's maximum is 2^8 above it (a probability is then below 2^8 and keeps its bits; a
                // published idea): following at once, half of the tiles of a few thousand keys rescale.
                if (__builtin_amdgcn_ballot_w64(mr * a.scale2 > m + 8.f) != 0) {
                    const float mx = fmax2(m, mr * a.scale2);
                    const float alpha = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mx);
                    m = mx;
                    l *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int reg = 0; reg < 16; ++reg) o[dt][reg] *= alpha;
                }
                const float nm = m == -INFINITY ? 0.f : -m;             // nothing seen so far: every exponent is -inf
                const float nf = far == 0.f ? nm : fmaf(far, a.scale2, nm);
                float xA[16], xB[16];
                float ls = 0.f;
#pragma unroll
                for (int reg = 0; reg < 16; ++reg) {
                    xA[reg] = __builtin_amdgcn_exp2f(fmaf(sA[reg], a.scale2, nf));
                    xB[reg] = __builtin_amdgcn_exp2f(fmaf(sB[reg], a.scale2, nf));
                    ls += xA[reg] + xB[reg];
                }
                l += half_sum(ls);
                const bf16x8_t pf[4] = {pack8(xA), pack8(xA + 8), pack8(xB), pack8(xB + 8)};
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[dt] = MFMA32(tr_frag<DP>(sV, dt, i, hh, r), pf[i], o[dt]);
                __builtin_amdgcn_s_setprio(0);
            }
            if (kp + 1 < np) {
                bits = key_bits(a, z, mk, kb + 64, lane);
                stage_commit<D, NTHR>(smem + ((kp + 1) & 1) * 2 * SC::TILE, sv, tid, bits);
            }
            __syncthreads();
        }
        {
            const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
            const bool ok = q < z.nq;
            const int64_t row = (int64_t)z.q0 + q;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if (l == 0.f) o[dt] = splat16(0.f);
                store_tile32(a.O + row * a.ldo + h * D + 32 * dt, o[dt], inv, hh, ok);
            }
            if (ok && a.lse && hh == 0) a.lse[(int64_t)h * a.Tq + row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
        }
        __syncthreads();                                                // the next tile of this block refills the first buffer
    }
}

// ------------------------------------------------------------------------------------------------ backward: dQ, delta, table gradient
// The forward's tiling with P recomputed from lse: dS = P (dO V^T - delta), dQ = scale dS K.
//
// TAB, the table's gradient: dtable[b] = sum of dS over a bucket's distances.  A row of dS sums to zero, so these sums cancel to a small part of
// their terms, and delta = rowsum(dO O) from the bf16 output would leave 2^-9 of it in them.  The walk over the keys therefore also sums dS by
// row: r = rowsum(P dP) - delta, the exact delta's distance from the rounded one (sum P = 1).  Tiles behind the last border are summed here, in
// compensated fp32, and corrected by r times their probability; the band of tiles around the diagonal is left to relattn_dkv_kernel, which has
// the exact delta.  Each block leaves its sums in its own row of `part`, added up in a fixed order by relattn_dtable_kernel.
// dQ and dK lose little by the rounded delta where many keys share a row; where a wave's queries see no more than one tile of keys, a first
// pass over the tile (already in LDS) takes the exact one.
// Bound like the forward (35 % of the cycles in the matrix units): 1.76 ms = 0.93 PFLOP/s without the table's gradient (16384 x 16 x 64), 2.00 ms with it; 0.39 / 0.42 ms (the documents).
// lse is one fp32 number: beyond 2^8 (in powers of two) its spacing leaves more than 2^-16 of a probability, at 1e6 five percent, at 1e8 nothing of log2(sum).
// Rows that far out sum their recomputed probabilities and divide by the sum: dQ (linear in P) at its end, dK / dV through RP::fix, a second term of the
// row's score.  Two sums, because the kernels round a score differently: here q.k joins the bias (as in the forward), there bias - lse.  Without
// such a row none of it is done: dQ asks per wave, dK / dV learns of it by a word per wave of dQ.  Costs of asking: backward with the table's gradient
// 152 -> 155 us (clips), 4.51 -> 4.54 ms (16384 x 16 x 64).
constexpr float BIG_LSE = 256.f;
constexpr int FAR_OUT = 1, LONE = 2;              // what a wave of dQ leaves for dK / dV: such a row, a sequence with at most one visible key
// dK / dV start a row's scores here, in units of the raw score
__device__ __forceinline__ float lse_start(float lse, float inv_scale) { return -lse * inv_scale; }
struct Comp {                                                           // compensated running sum
    float s = 0.f, c = 0.f;
    __device__ __forceinline__ void add(float v) {
        const float y = v - c, t = s + y;
        c = (t - s) - y;
        s = t;
    }
};
template <int D, int NW, bool TAB>
__global__ void __launch_bounds__(NW * 64, D <= 32 ? 3 : 2) relattn_dq_kernel(RP a) {
    constexpr int KS = D / 16, DT = D / 32, DP = D + 8, NTHR = NW * 64;
    constexpr bool SPLIT = D >= 96;
    using SC = StageC<D, NTHR>;
    extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
    const int blen = bias_len(a.far, a.causal);
    float* bv = reinterpret_cast<float*>(smem + 4 * SC::TILE);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // (wave-uniform for the compiler too)
    const int r = lane & 31, hh = lane >> 5;
    const Who w = who(a, a.H);
    const int h = w.h, hk = h / (a.H / a.Hkv);
    if (w.s == a.S) {
        const int64_t from = tail_start(a.cu_q, a.S, a.Tq);
        zero_rows(a.dQ, a.lddq, from, a.Tq, h * D, D, a.tiles * NTHR, w.tile * NTHR + tid);
        return;
    }
    const Seq z = seq_of(a, w.s);
    const int shift = z.nk - z.nq;
    fill_bias(a, h, bv, tid, NTHR);
    Stage<D, NTHR> sg;
    sg.plan(tid, a.ldk, a.ldv);
    float tab_l = 0.f, tab_r = 0.f;                                     // the lane's sums behind the borders, corrected
    int saw = 0;
    uint32_t* word = a.seen + (((int64_t)w.s * a.H + h) * a.tiles + w.tile) * NW + wave;
    if ((int64_t)w.tile * 32 * NW >= z.nq && lane == 0) word[0] = 0;
    __syncthreads();
    const float cleft = bv[0], cright = bv[blen - 1];
    for (int64_t tile = w.tile; tile * 32 * NW < z.nq; tile += a.tiles) {
        const int nt = (z.nq + 32 * NW - 1) / (32 * NW);
        const int qt = a.causal ? nt - 1 - (int)tile : (int)tile;
        const int qb = qt * 32 * NW, qw = qb + 32 * wave;
        const bool live = qw < z.nq;
        const int q = qw + r;
        const bool qok = q < z.nq;
        const int64_t qrow = (int64_t)z.q0 + (qok ? q : z.nq - 1);
        const int plo = qw + shift, phi = plo + 31, pos = plo + r;
        bf16x8_t qf[KS], df[KS];
        float delta = 0.f;
        {
            const bf16_t* qp = a.Q + qrow * a.ldq + h * D + 8 * hh;
            const bf16_t* dp = a.dO + qrow * a.lddo + h * D + 8 * hh;
            const bf16_t* op = a.O + qrow * a.ldo + h * D + 8 * hh;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[s] = ld_frag(qp + 16 * s);
                df[s] = ld_frag(dp + 16 * s);
                const bf16x8_t of = ld_frag(op + 16 * s);
#pragma unroll
                for (int j = 0; j < 8; ++j) delta += bf2f((bf16_t)df[s][j]) * bf2f((bf16_t)of[j]);
            }
        }
        delta = half_sum(delta);
        const float lse = a.lse[(int64_t)h * a.Tq + qrow];
        const bool seen = qok && lse != -INFINITY;                      // a row that saw no key has no gradient
        const float nl = seen ? -lse * LOG2E : -INFINITY;
        if (!seen) delta = 0.f;
        const bool big = seen && fabsf(nl) > BIG_LSE;
        const bool sums = __builtin_amdgcn_ballot_w64(big) != 0;        // some row of the wave needs its sum
        float psum = 0.f, ksum = 0.f;                                   // the lane's share of it, as here and as dK / dV add bias, lse and q.k
        f32x16_t dq[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dq[dt] = splat16(0.f);
        int kend = z.nk;
        if (a.causal) {
            const int last = qb + 32 * NW + shift;
            kend = kend < last ? kend : (last < 0 ? 0 : last);
        }
        const int np = (kend + 63) >> 6;
        const bf16_t* Kb = a.K + (int64_t)z.k0 * a.ldk + hk * D;
        const bf16_t* Vb = a.V + (int64_t)z.k0 * a.ldv + hk * D;
        Comp all, sl, sr;                                               // the lane's share of its row: sum dS, behind the left / right border
        float br = 0.f, bn = 0.f;                                       // probability behind the right border, around the diagonal
        // Wide heads: K and V take turns in one half's staging registers (K arrives behind the first 32 keys' products, V behind the second's), which
        // leaves room for two waves per SIMD.
        u32x4_t sv[SPLIT ? SC::HALF : SC::PER];
        uint64_t bits = 0, nbits = 0;
        int mk = 0;
        if (np > 0) {
            mk = key_load(a, z, 0, lane);
            if constexpr (SPLIT) {
                sg.fetch1(sv, tid, Kb, a.ldk, 0, 0, z.nk);
                bits = key_bits(a, z, mk, 0, lane);
                commit_one<D, NTHR>(smem, sv, tid, bits);
                sg.fetch1(sv, tid, Vb, a.ldv, 1, 0, z.nk);
                commit_one<D, NTHR>(smem + SC::TILE, sv, tid, bits);
            } else {
                sg.fetch(sv, tid, Kb, a.ldk, Vb, a.ldv, 0, z.nk);
                bits = key_bits(a, z, mk, 0, lane);
                stage_commit<D, NTHR>(smem, sv, tid, bits);
            }
        }
        __syncthreads();
        arrived(qf);
        arrived(df);
        saw |= (sums ? FAR_OUT : 0) | (few(bits) && lone_key(a, z, lane) ? LONE : 0);
        if (lane == 0) word[0] = saw;
        auto visible = [&](int kb, uint64_t in) -> uint64_t {           // the keys of a tile that the lane's query sees, from its half-wave's first on
            if (a.causal) {
                const int c = pos - kb;
                in = c < 0 ? 0 : (c >= 63 ? in : in & ((2ull << c) - 1));
            }
            return in >> (4 * hh);
        };
        const int span = a.causal && phi < z.nk ? phi + 1 : z.nk;       // keys the wave's queries see at most
        if (live && bits != 0 && span > 0 && span <= 64) {              // few keys: delta = rowsum(P dP) first (see above)
            float t = 0.f, l = 0.f;
            const uint64_t vis = visible(0, bits);
            const bool left = 63 - plo <= -a.far, right = -phi >= a.far;
            const float nf = left || right ? fmaf(left ? cleft : cright, a.scale2, nl) : nl;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                const bf16_t* tK = smem + half * 32 * DP;
                f32x16_t sc = splat16(0.f), dp = splat16(0.f);
                if (!left && !right) sc = bias16(bv, 4 * hh - pos + a.far + PAD + 32 * half);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    sc = MFMA32(nat_frag<DP>(tK, r, hh, s), qf[s], sc);
                    dp = MFMA32(nat_frag<DP>(tK + SC::TILE, r, hh, s), df[s], dp);
                }
#pragma unroll
                for (int reg = 0; reg < 16; ++reg) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(sc[reg], a.scale2, nf));
                    const bool on = (vis >> (32 * half + ACC_ROW(reg, 0))) & 1;
                    l += on ? e : 0.f;
                    t += on ? e * dp[reg] : 0.f;
                }
            }
            t = half_sum(t);
            l = half_sum(l);
            delta = l > 0.f ? t / l : 0.f;
        }
        // dP - delta: the accumulator starts at -delta, 16 registers held for that where there is room (D <= 64), else a subtraction
        constexpr bool HOLD = D <= 64;
        const f32x16_t ndel = splat16(HOLD ? -delta : 0.f);
        for (int kp = 0; kp < np; ++kp) {
            const bf16_t* sK = smem + (kp & 1) * 2 * SC::TILE;
            const bf16_t* sV = sK + SC::TILE;
            const int kb = 64 * kp;
            if (kp + 1 < np) {
                mk = key_load(a, z, kb + 64, lane);
                if constexpr (SPLIT) sg.fetch1(sv, tid, Kb, a.ldk, 0, kb + 64, z.nk);
                else sg.fetch(sv, tid, Kb, a.ldk, Vb, a.ldv, kb + 64, z.nk);
            }
            bf16_t* nK = smem + ((kp + 1) & 1) * 2 * SC::TILE;
            const bool left = kb + 63 - plo <= -a.far, right = kb - phi >= a.far;
            const bool act = live && bits != 0 && !(a.causal && kb > phi);
            {
                const int idx0 = kb + 4 * hh - pos + a.far + PAD;
                const uint64_t vis = visible(kb, bits);
                const bool edge = bits != ~0ull || (a.causal && kb + 63 > plo);
                const float nf = left || right ? fmaf(left ? cleft : cright, a.scale2, nl) : nl;
                if (sums && act) {                                  // (apart from the products below, whose registers it would lengthen)
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        const float first = lse_start(a.lse[(int64_t)h * a.Tq + qrow], a.inv_scale);
                        f32x16_t sc = splat16(0.f), sk = splat16(first + (left ? cleft : cright));
                        if (!left && !right) {
                            sc = bias16(bv, idx0 + 32 * half);
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) sk[reg] = first + sc[reg];
                        }
#pragma unroll
                        for (int s = 0; s < KS; ++s) {
                            const bf16x8_t kf = nat_frag<DP>(sK + half * 32 * DP, r, hh, s);
                            sc = MFMA32(kf, qf[s], sc);
                            sk = MFMA32(kf, qf[s], sk);
                        }
#pragma unroll
                        for (int reg = 0; reg < 16; ++reg) {
                            const bool on = (vis >> (32 * half + ACC_ROW(reg, 0))) & 1;
                            const float e = __builtin_amdgcn_exp2f(fmaf(sc[reg], a.scale2, nf)), f = __builtin_amdgcn_exp2f(sk[reg] * a.scale2);
                            psum += on ? e : 0.f;
                            ksum += on ? f : 0.f;
                        }
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {              // the two 32-key tiles, one after the other (register budget)
                    if (act) {
                        const bf16_t* tK = sK + half * 32 * DP;
                        const bf16_t* tV = sV + half * 32 * DP;
                        const int idx = idx0 + 32 * half;
                        f32x16_t sc, dp = MFMA32(nat_frag<DP>(tV, r, hh, 0), df[0], ndel);
                        if (left || right) sc = MFMA32(nat_frag<DP>(tK, r, hh, 0), qf[0], splat16(0.f));
                        else sc = MFMA32(nat_frag<DP>(tK, r, hh, 0), qf[0], bias16(bv, idx));
#pragma unroll
                        for (int s = 1; s < KS; ++s) {
                            sc = MFMA32(nat_frag<DP>(tK, r, hh, s), qf[s], sc);
                            dp = MFMA32(nat_frag<DP>(tV, r, hh, s), df[s], dp);
                        }
                        float p[16], ds[16];
#pragma unroll
                        for (int reg = 0; reg < 16; ++reg) {
                            p[reg] = __builtin_amdgcn_exp2f(fmaf(sc[reg], a.scale2, nf));
                            ds[reg] = p[reg] * (HOLD ? dp[reg] : dp[reg] - delta);
                        }
                        if (edge) {
                            asm volatile("");                           // (kept a branch: as selects these run in every tile)
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) {
                                const bool on = (vis >> (32 * half + ACC_ROW(reg, 0))) & 1;
                                p[reg] = on ? p[reg] : 0.f;
                                ds[reg] = on ? ds[reg] : 0.f;
                            }
                        }
                        if (TAB) {
                            float t = 0.f;
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) t += ds[reg];
                            all.add(t);
                            if (left) sl.add(t);
                            if (right) sr.add(t);
                            if (!left) {                            // the probability behind the left border is what is left of one
                                float b = 0.f;
#pragma unroll
                                for (int reg = 0; reg < 16; ++reg) b += p[reg];
                                if (right) br += b; else bn += b;
                            }
                        }
                        const bf16x8_t d0 = pack8(ds), d1 = pack8(ds + 8);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            dq[dt] = MFMA32(tr_frag<DP>(tK, dt, 0, hh, r), d0, dq[dt]);
                            dq[dt] = MFMA32(tr_frag<DP>(tK, dt, 1, hh, r), d1, dq[dt]);
                        }
                    }
                    if constexpr (SPLIT) {
                        if (half == 0 && kp + 1 < np) {
                            nbits = key_bits(a, z, mk, kb + 64, lane);
                            commit_one<D, NTHR>(nK, sv, tid, nbits);
                            sg.fetch1(sv, tid, Vb, a.ldv, 1, kb + 64, z.nk);
                        }
                    }
                }
            }
            if (kp + 1 < np) {
                if constexpr (SPLIT) {
                    commit_one<D, NTHR>(nK + SC::TILE, sv, tid, nbits);
                    bits = nbits;
                } else {
                    bits = key_bits(a, z, mk, kb + 64, lane);
                    stage_commit<D, NTHR>(nK, sv, tid, bits);
                }
            }
            __syncthreads();
        }
        float norm = 1.f;                                               // of a row far out: 1 / sum P; dK / dV's second term goes to a.fix
        if (sums) {
            psum = half_sum(psum);
            ksum = half_sum(ksum);
            if (big && psum > 0.f) norm = 1.f / psum;
            if (big && hh == 0) a.fix[(int64_t)h * a.Tq + qrow] = ksum > 0.f ? -__log2f(ksum) / a.scale2 : 0.f;
        }
        const bool lone = (saw & LONE) != 0;
        bf16_t* dqp = a.dQ + ((int64_t)z.q0 + q) * a.lddq + h * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) store_tile32(dqp + 32 * dt, dq[dt], lone ? 0.f : a.scale * norm, hh, qok);
        if (TAB && !lone) {
            const float rs = half_sum(all.s - all.c) * norm;
            br = half_sum(br) * norm;
            bn = half_sum(bn) * norm;
            const float bl = fmaxf(1.f - br - bn, 0.f);
            if (hh == 0 && seen) {                                      // once per row: the halves' sums of dS enter below, one per lane
                tab_l -= rs * bl;
                tab_r -= rs * br;
            }
            delta += rs;                                                // rowsum(P dP) to fp32
            tab_l += (sl.s - sl.c) * norm;
            tab_r += (sr.s - sr.c) * norm;
        }
        if (qok && hh == 0) a.delta[(int64_t)h * a.Tq + qrow] = delta;
    }
    if (TAB) {
        tab_l = wave_sum<64>(tab_l);
        tab_r = wave_sum<64>(tab_r);
        __syncthreads();
        if (lane == 0) { bv[2 * wave] = tab_l; bv[2 * wave + 1] = tab_r; }
        __syncthreads();
        if (tid < 2) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) t += bv[2 * w + tid];
            a.part[(((int64_t)w.s * a.tiles + w.tile) * a.H + h) * 2 + tid] = t;
        }
    }
}

// dtable[b][h] = sum of the band's rows, and of the rows behind the borders where b is a side's last bucket, in order
__global__ void __launch_bounds__(256) relattn_dtable_kernel(const float* band, int nband, const float* behind, int nbehind, float* dtable, int H, int NB, int causal) {
    __shared__ float s[256];
    const int h = blockIdx.x, b = blockIdx.y;
    float t = 0.f;
    for (int i = threadIdx.x; i < nband; i += 256) t += band[((int64_t)i * H + h) * NB + b];
    const int left = causal ? NB - 1 : NB / 2 - 1;
    if (b == left || b == NB - 1)
        for (int i = threadIdx.x; i < nbehind; i += 256) t += behind[((int64_t)i * H + h) * 2 + (b == left ? 0 : 1)];
    s[threadIdx.x] = t;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) s[threadIdx.x] += s[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) dtable[(int64_t)b * H + h] = s[0];
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV
// A block = one (sequence, key / value head) and 32 NW keys, 32 per wave; it walks the queries of every head of the group in 64-row tiles
// of Q and dO, so the gradients of a shared head are summed in registers, in one order.  S[q][key]: rows = queries, lane = key.
//
// TAB: the table's gradient of the tiles that relattn_dq_kernel does not count as lying behind a border; delta is the exact one by now.  A tile of dS goes
// through 32 LDS rows of 33 (no bank conflicts) and lane l adds up its diagonals: column c of row (c + 31 - l) mod 32 belongs to the distance
// base - 31 + l for c <= l, to base + 1 + l behind it (base = key - query of the tile's corner).  The next 32 queries lie 32 below: their upper
// diagonals complete this tile's lower ones, so every 32 queries a wave adds 32 finished sums to an LDS array by distance.  Two arrays, of the even
// and the odd waves: waves two apart touch distances 64 apart, and a barrier lies between two steps, so no addition meets another and
// the order is fixed.  After each head the arrays fold into the buckets, a row of `part` per block.  (A kernel of its own for the band that computed
// scores and dS again took 60 us where this adds 35 us, 32 clips of 131 .. 490 x 12 x 64; LDS additions per element 340 us.)
// 2.17 ms = 1.01 PFLOP/s without the table's gradient (16384 x 16 x 64), 2.41 ms with it (distances up to 800); 0.65 / 0.75 ms (the documents, whose 492
// registers leave one wave per SIMD: the walk waits for its own LDS reads.  Two waves per SIMD spilled, 2.6 ms, or, as eight waves with the keys in LDS
// and half a tile's queries each, read a quarter more from LDS: the whole backward 1.19 ms against 1.07 without the table).
constexpr int STATS = 2 * (5 * 64 + 4);           // 5 x 64 floats and the waves' votes, in bf16 elements
template <int D, int NW, bool TAB>
__global__ void __launch_bounds__(NW * 64, D <= 64 ? 2 : 1) relattn_dkv_kernel(RP a) {
    constexpr int KS = D / 16, DT = D / 32, DP = D + 8, NTHR = NW * 64;
    constexpr bool WIDE = D >= 96;
    using SC = StageC<D, NTHR>;
    constexpr int BUF = 2 * SC::TILE + STATS;                           // Q and dO tiles and their rows' statistics
    extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
    float* bv = reinterpret_cast<float*>(smem + 2 * BUF);
    const int blen = bias_len(a.far, a.causal), alen = (blen + 3) & ~3;
    float* by = bv + alen;                                              // TAB: [2][alen] sums by distance, [NW][32][33] tiles, [alen] bucket ids
    float* skew = by + 2 * alen;
    uint8_t* ids = reinterpret_cast<uint8_t*>(skew + NW * 32 * 33);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // (wave-uniform for the compiler too)
    const int r = lane & 31, hh = lane >> 5;
    const Who w = who(a, a.Hkv * a.hsplit);
    const int hk = w.h / a.hsplit, rep = a.H / a.Hkv / a.hsplit, head0 = w.h * rep;       // the block's heads: head0 .. head0 + rep - 1
    if (w.s == a.S) {
        const int64_t from = tail_start(a.cu_k, a.S, a.Tk);
        const int step = a.tiles * NTHR, off = w.tile * NTHR + tid;
        zero_rows(a.dK, a.lddk, from, a.Tk, hk * D, D, step, off);
        zero_rows(a.dV, a.lddv, from, a.Tk, hk * D, D, step, off);
        return;
    }
    const Seq z = seq_of(a, w.s);
    const int shift = z.nk - z.nq;
    float* rows = TAB ? a.part + (((int64_t)w.s * a.tiles + w.tile) * a.H + head0) * a.NB + tid : nullptr;
    if (TAB) {
        for (int i = tid; i < alen; i += NTHR) {
            int x = i - (a.far + PAD);
            x = x < -a.far ? -a.far : (x > a.far ? a.far : x);
            ids[i] = (uint8_t)a.plan[x + a.far];
        }
        for (int g = 0; g < rep && tid < a.NB; ++g) rows[(int64_t)g * a.NB] = 0.f;
    }
    uint32_t* vote = reinterpret_cast<uint32_t*>(smem + 2 * SC::TILE) + 320;      // (in the first buffer's statistics)
    uint32_t any = 0;                                                   // what dQ saw among this block's heads
    {
        const int n = rep * a.qtiles * 4;
        const uint32_t* seen = a.seen + ((int64_t)w.s * a.H + head0) * a.qtiles * 4;
        if (tid < n) any = seen[tid];
        for (int i = tid + NTHR; i < n; i += NTHR) any |= seen[i];
    }
    auto votes = [&]() -> int { return __builtin_amdgcn_readfirstlane(vote[0] | vote[1] | vote[2] | vote[3]); };
    Stage<D, NTHR> sg;
    sg.plan(tid, a.ldq, a.lddo);
    for (int64_t tile = w.tile; tile * 32 * NW < z.nk; tile += a.tiles) {
        const int kw = 32 * ((int)tile * NW + wave);
        const int key = kw + r;
        bool kok = key < z.nk;
        const int64_t krow = (int64_t)z.k0 + (kok ? key : z.nk - 1);
        const bool stored = kok;
        if (a.kmask != nullptr && kok) kok = a.kmask[krow] != 0;
        const bool live = __builtin_amdgcn_ballot_w64(kok) != 0;
        bf16x8_t kf[KS], vf[KS];
        {
            const bf16_t* kp = a.K + krow * a.ldk + hk * D + 8 * hh;
            const bf16_t* vp = a.V + krow * a.ldv + hk * D + 8 * hh;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                kf[s] = ld_frag(kp + 16 * s);
                vf[s] = ld_frag(vp + 16 * s);
                if (!kok) { kf[s] = zero_frag(); vf[s] = zero_frag(); }
            }
        }
        f32x16_t dk[DT], dv[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) { dk[dt] = splat16(0.f); dv[dt] = splat16(0.f); }
        // first query that may see the block's first key
        int qfirst = a.causal ? (int)tile * 32 * NW - shift : 0;
        qfirst = qfirst < 0 ? 0 : qfirst;
        const int p0 = qfirst >> 6, np = (z.nq + 63) >> 6;
        arrived(kf);
        arrived(vf);
        if (tile == w.tile) {
            const uint64_t far_out = __builtin_amdgcn_ballot_w64((any & FAR_OUT) != 0), lone = __builtin_amdgcn_ballot_w64((any & LONE) != 0);
            if (lane == 0) vote[wave] = (far_out != 0 ? FAR_OUT : 0) | (lone != 0 ? LONE : 0);
            any = 0;
        }
        for (int g = 0; g < rep && p0 < np; ++g) {
            const int h = head0 + g;
            const bf16_t* Qb = a.Q + (int64_t)z.q0 * a.ldq + h * D;
            const bf16_t* Db = a.dO + (int64_t)z.q0 * a.lddo + h * D;
            const float* lseb = a.lse + (int64_t)h * a.Tq + z.q0;
            const float* delb = a.delta + (int64_t)h * a.Tq + z.q0;
            const float* fixb = a.fix + (int64_t)h * a.Tq + z.q0;
            u32x4_t sv[SC::PER];
            float nl = 0.f, nd = 0.f, cleft, cright;
            auto fetch_all = [&](int q0) {
                sg.fetch(sv, tid, Qb, a.ldq, Db, a.lddo, q0, z.nq);
                if (tid < 64) {
                    const int qi = q0 + tid < z.nq ? q0 + tid : z.nq - 1;
                    nl = lseb[qi];
                    nd = delb[qi];
                }
            };
            auto commit_all = [&](bf16_t* buf, int q0, int apart) {
                const int left = z.nq - q0;
                stage_commit<D, NTHR>(buf, sv, tid, left >= 64 ? ~0ull : (1ull << left) - 1);
                float* st = reinterpret_cast<float*>(buf + 2 * SC::TILE);
                if (tid < 64) {                                         // lse in units of the raw score; a row that saw nothing, or none at all: P = 0
                    const bool ok = tid < left && nl != -INFINITY;
                    const float l = ok ? lse_start(nl, a.inv_scale) : -INFINITY;
                    st[tid] = l;
                    st[64 + tid] = l + cleft;
                    st[128 + tid] = l + cright;
                    st[192 + tid] = ok ? -nd : 0.f;
                    if (apart != 0) {                                   // the second term: behind a border it joins the sum
                        const float f = ok && fabsf(nl * LOG2E) > BIG_LSE ? fixb[q0 + tid] : 0.f;
                        st[64 + tid] = (l + cleft) + f;
                        st[128 + tid] = (l + cright) + f;
                        st[256 + tid] = f;
                    }
                }
            };
            fetch_all(64 * p0);
            fill_bias(a, h, bv, tid, NTHR);
            if (TAB)
                for (int i = tid; i < 2 * alen; i += NTHR) by[i] = 0.f;
            float* mine = by + (wave & 1) * alen + a.far + PAD + r;         // the wave's array, by distance
            float* m = skew + wave * 32 * 33;
            float prev = 0.f;                                           // lane l: sum of distance prev_base - 31 + l, still open
            int prev_base = 0;
            bool open = false;
            auto close = [&](int at, float v) {                         // 32 finished sums, of distances at .. at + 31
                if (hh == 0) mine[at] += v;
            };
            __syncthreads();
            cleft = bv[0];
            cright = bv[blen - 1];
            int apart = votes() & FAR_OUT;
            commit_all(smem + (p0 & 1) * BUF, 64 * p0, apart);
            __syncthreads();
            for (int qp = p0; qp < np; ++qp) {
                const bf16_t* sQ = smem + (qp & 1) * BUF;
                const bf16_t* sD = sQ + SC::TILE;
                const float* sL = reinterpret_cast<const float*>(sQ + 2 * SC::TILE);
                if (qp + 1 < np) fetch_all(64 * (qp + 1));
                const int pb = 64 * qp + shift;                         // position of the tile's first query
                asm volatile("" : "+s"(apart));                         // (else the walk is compiled twice, and spills)
                if (live && !(a.causal && pb + 63 < kw)) {
                    const bool left = kw + 31 - pb <= -a.far, right = kw - (pb + 63) >= a.far;
                    const bool edge = a.causal && kw + 31 > pb;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const bf16_t* tQ = sQ + half * 32 * DP;
                        const bf16_t* tD = sD + half * 32 * DP;
                        const int rel = key - (pb + 32 * half) - 4 * hh;    // distance of accumulator row 0
                        // the accumulators start at bias - lse (behind a border the two were added once per query) and at -delta
                        f32x16_t sc, dp;
                        const float* st = sL + 64 * (left ? 1 : (right ? 2 : 0)) + 32 * half + 4 * hh;
#pragma unroll
                        for (int g4 = 0; g4 < 4; ++g4) {
                            const float4 ls = *reinterpret_cast<const float4*>(st + 8 * g4);
                            const float4 de = *reinterpret_cast<const float4*>(sL + 192 + 32 * half + 8 * g4 + 4 * hh);
                            sc[4 * g4] = ls.x; sc[4 * g4 + 1] = ls.y; sc[4 * g4 + 2] = ls.z; sc[4 * g4 + 3] = ls.w;
                            dp[4 * g4] = de.x; dp[4 * g4 + 1] = de.y; dp[4 * g4 + 2] = de.z; dp[4 * g4 + 3] = de.w;
                        }
                        if (!left && !right) {
                            asm volatile("");
                            const float* bp = bv + rel + a.far + PAD;
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) sc[reg] += bp[-ACC_ROW(reg, 0)];
                            if (apart != 0) {
                                asm volatile("");
                                const float* fx = sL + 256 + 32 * half + 4 * hh;
#pragma unroll
                                for (int reg = 0; reg < 16; ++reg) sc[reg] += fx[ACC_ROW(reg, 0)];
                            }
                        }
                        // one wave per SIMD (D >= 96): nothing else hides the LDS latency, so the operands of a whole phase are asked for at once
                        bf16x8_t qa[KS], da[KS];
#pragma unroll
                        for (int s = 0; s < KS; ++s) { qa[s] = nat_frag<DP>(tQ, r, hh, s); da[s] = nat_frag<DP>(tD, r, hh, s); }
                        if (WIDE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int s = 0; s < KS; ++s) {
                            sc = MFMA32(qa[s], kf[s], sc);
                            dp = MFMA32(da[s], vf[s], dp);
                        }
                        bf16x8_t to[2][4];                              // transposed operands of one 32-column block: dO, dO, Q, Q
                        auto trans = [&](int dt) {
                            to[dt & 1][0] = tr_frag<DP>(tD, dt, 0, hh, r); to[dt & 1][1] = tr_frag<DP>(tD, dt, 1, hh, r);
                            to[dt & 1][2] = tr_frag<DP>(tQ, dt, 0, hh, r); to[dt & 1][3] = tr_frag<DP>(tQ, dt, 1, hh, r);
                        };
                        if (WIDE) { trans(0); __builtin_amdgcn_sched_barrier(0); }
                        float pr[16], ds[16];
#pragma unroll
                        for (int reg = 0; reg < 16; ++reg) {
                            const float p = __builtin_amdgcn_exp2f(sc[reg] * a.scale2);
                            pr[reg] = p;
                            ds[reg] = p * dp[reg];
                        }
                        if (edge) {                                     // hidden by the causal rule (dS too, whatever dP holds)
                            asm volatile("");                           // (kept a branch: as selects these run in every tile)
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) {
                                pr[reg] = rel <= ACC_ROW(reg, 0) ? pr[reg] : 0.f;
                                ds[reg] = rel <= ACC_ROW(reg, 0) ? ds[reg] : 0.f;
                            }
                        }
                        const int plo = pb + 32 * half, kb = kw & ~63;
                        const bool near = TAB && kb + 63 - plo > -a.far && kb - plo - 31 < a.far && !(a.causal && kw > plo + 31);
                        if (near) {
#pragma unroll
                            for (int reg = 0; reg < 16; ++reg) m[(ACC_ROW(reg, 0) + 4 * hh) * 33 + r] = kok ? ds[reg] : 0.f;
                            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                            float lo = 0.f, all = 0.f;
                            int at = (31 - r) * 33 + 16 * 34 * hh;      // column 16 hh of the lane's lower diagonal; the upper one 32 rows back
                            int behind = r - 16 * hh;
                            asm volatile("" : "+v"(at), "+v"(behind));  // (else the sixteen addresses are kept, and spilled, across the walk)
                            const float* m0 = m + at;
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                const bool up = c > behind;
                                const float v = (up ? m0 - 32 * 33 : m0)[34 * c];
                                lo += up ? 0.f : v;
                                all += v;
                            }
                            const float hi = half_sum(all - lo);
                            const int base = kw - plo;
                            close(base + 1, open ? hi + prev : hi);
                            prev = half_sum(lo);
                            prev_base = base;
                            open = true;
                        } else if (TAB && open) {
                            close(prev_base - 31, prev);
                            open = false;
                        }
                        const bf16x8_t a0 = pack8(pr), a1 = pack8(pr + 8), d0 = pack8(ds), d1 = pack8(ds + 8);
                        if (!WIDE) trans(0);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            if (dt + 1 < DT) trans(dt + 1);
                            if (WIDE) __builtin_amdgcn_sched_barrier(0);
                            dv[dt] = MFMA32(to[dt & 1][0], a0, dv[dt]);
                            dk[dt] = MFMA32(to[dt & 1][2], d0, dk[dt]);
                            dv[dt] = MFMA32(to[dt & 1][1], a1, dv[dt]);
                            dk[dt] = MFMA32(to[dt & 1][3], d1, dk[dt]);
                        }
                    }
                }
                if (qp + 1 < np) commit_all(smem + ((qp + 1) & 1) * BUF, 64 * (qp + 1), apart);
                __syncthreads();
            }
            if (TAB && !(votes() & LONE)) {                             // a thread per bucket and slice of the distances, then the slices in order
                if (open) close(prev_base - 31, prev);
                __syncthreads();
                const int nb2 = 1 << (32 - __builtin_clz(a.NB - 1)), sl = NTHR / nb2, b = tid & (nb2 - 1);
                const int n4 = alen / 4, per = (n4 + sl - 1) / sl, from = tid / nb2 * per, to = min(from + per, n4);
                float t = 0.f;
#pragma unroll 2
                for (int i = from; i < to; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(by + 4 * i), y = *reinterpret_cast<const float4*>(by + alen + 4 * i);
                    const uint32_t id = *reinterpret_cast<const uint32_t*>(ids + 4 * i);
                    t += (int)(id & 255) == b ? x.x + y.x : 0.f;
                    t += (int)(id >> 8 & 255) == b ? x.y + y.y : 0.f;
                    t += (int)(id >> 16 & 255) == b ? x.z + y.z : 0.f;
                    t += (int)(id >> 24) == b ? x.w + y.w : 0.f;
                }
                skew[tid] = t;
                __syncthreads();
                if (tid < a.NB) {
                    for (int i = 1; i < sl; ++i) t += skew[i * nb2 + tid];
                    rows[(int64_t)g * a.NB] += t;
                }
                __syncthreads();
            }
        }
        const bool lone = p0 < np && (votes() & LONE);
        if (a.hsplit > 1) {
            const int64_t n = a.Tk * a.Hkv * D;
            float* kp = a.pk + 2 * (w.h - hk * a.hsplit) * n + (((int64_t)z.k0 + key) * a.Hkv + hk) * D + 4 * hh;
            if (stored) {
                const float sk = kok && !lone ? a.scale : 0.f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const int c = 32 * dt + 8 * g4;
                        float x[4], y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {                   // (a masked key's sums may be anything)
                            x[j] = kok ? dk[dt][4 * g4 + j] * sk : 0.f;
                            y[j] = kok ? dv[dt][4 * g4 + j] : 0.f;
                        }
                        *reinterpret_cast<float4*>(kp + c) = make_float4(x[0], x[1], x[2], x[3]);
                        *reinterpret_cast<float4*>(kp + n + c) = make_float4(y[0], y[1], y[2], y[3]);
                    }
            }
            __syncthreads();
            continue;
        }
        bf16_t* kp = a.dK + ((int64_t)z.k0 + key) * a.lddk + hk * D;
        bf16_t* vp = a.dV + ((int64_t)z.k0 + key) * a.lddv + hk * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if (!kok) { dk[dt] = splat16(0.f); dv[dt] = splat16(0.f); }     // a masked key has no gradient
            store_tile32(kp + 32 * dt, dk[dt], lone ? 0.f : a.scale, hh, stored);
            store_tile32(vp + 32 * dt, dv[dt], 1.0f, hh, stored);
        }
        __syncthreads();
    }
}

// dK and dV from the parts of the blocks that shared a key / value head's query heads, summed in order; rows behind the last sequence as in zero_tail
__global__ void __launch_bounds__(256) relattn_kvsum_kernel(RP a, int kd) {
    const int per = kd / 4;
    const int64_t n = a.Tk * kd, from = tail_start(a.cu_k, a.S, a.Tk);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.Tk * per; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per;
        const int col = 4 * (int)(i - row * per);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (row < from) {
            const float* p = a.pk + row * kd + col;
            for (int k = 0; k < a.hsplit; ++k, p += 2 * n) {
                const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + n);
                x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
                y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
            }
        } else if (!a.zero_tail) continue;
        *reinterpret_cast<uint2*>(a.dK + row * a.lddk + col) = make_uint2(pack_bf2(x.x, x.y), pack_bf2(x.z, x.w));
        *reinterpret_cast<uint2*>(a.dV + row * a.lddv + col) = make_uint2(pack_bf2(y.x, y.y), pack_bf2(y.z, y.w));
    }
}

// ------------------------------------------------------------------------------------------------ one new token per sequence
struct DP_ {
    const bf16_t* Q; int64_t ldq;
    const bf16_t* K; int64_t ldk, bsk;
    const bf16_t* V; int64_t ldv, bsv;
    bf16_t* O; int64_t ldo;
    const int32_t* lens;
    int S, cap, H, Hkv;
    const float* table; const int32_t* plan;
    int NB, far;
    float scale2, inv_scale;
    int chunk, nsplit;
    float* po;                        // [S, nsplit, H, D] partial outputs (normalised by their own sum)
    float* pl;                        // [S, nsplit, H] log2-domain lse of the part, -inf when empty
};

// A block = `chunk` keys of one (sequence, key / value head) against all query heads of the group: the heads are the 32 columns of the
// MFMA (unused columns are zero), so a key or value row is read once whatever the group's size.  Each of the four waves walks its own
// 32-key tiles with its own LDS tile (no barrier in the loop), the next tile's 16-byte pieces in flight meanwhile; the waves' statistics
// meet in LDS at the end.  Bound by the bytes of K and V: 538 MB in 131 us = 4.1 TB/s (64 sequences of 1 .. 4096, 8 heads of 128), 1.40 GB in 272 us =
// 5.1 TB/s (8 of 20011 .. 65536); one sequence of 701 takes two launches of 8 + 3 us, all latency.
template <int D>
__global__ void __launch_bounds__(256, 2) relattn_decode_kernel(DP_ a) {
    constexpr int KS = D / 16, DT = D / 32, DP = D + 8, ROWP = D / 8, PER = 2 * 32 * ROWP / 64, TILE = 32 * DP;
    extern __shared__ __attribute__((aligned(16))) bf16_t smem[];       // per wave {K, V} x [32][DP]; then the table's columns [NB][32]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // (wave-uniform for the compiler too)
    const int r = lane & 31, hh = lane >> 5;
    const int rep = a.H / a.Hkv, ncg = (rep + 31) / 32;
    const int hk = blockIdx.y / ncg, cg = blockIdx.y - hk * ncg;
    const int ncol = rep - 32 * cg < 32 ? rep - 32 * cg : 32;
    const int h0 = hk * rep + 32 * cg;                                  // head of column 0
    const int s = blockIdx.z, sp = blockIdx.x;
    int len = a.lens[s];
    len = len < 0 ? 0 : (len > a.cap ? a.cap : len);
    const int k0 = sp * a.chunk, k1 = k0 + a.chunk < len ? k0 + a.chunk : len;
    if (k0 >= len && sp > 0) return;                                    // the combining pass knows which parts exist
    const int pos = len - 1;
    const bf16_t* Kb = a.K + (int64_t)s * a.bsk + hk * D;
    const bf16_t* Vb = a.V + (int64_t)s * a.bsv + hk * D;
    bf16_t* sK = smem + wave * 2 * TILE;
    bf16_t* sV = sK + TILE;
    float* sb = reinterpret_cast<float*>(smem + 8 * TILE);              // [NB][32] table columns in raw score units
    const bool col = r < ncol;
    u32x4_t sv[PER];
    auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int id = lane + 64 * i;
            const int which = id / (32 * ROWP), rem = id - which * 32 * ROWP;
            const int rr = rem / ROWP, c = rem - rr * ROWP;
            int row = kb + rr;
            row = row < k1 ? row : k1 - 1;
            sv[i] = *reinterpret_cast<const u32x4_t*>((which ? Vb + (int64_t)row * a.ldv : Kb + (int64_t)row * a.ldk) + 8 * c);
        }
    };
    int kb = k0 + 32 * wave;
    if (kb < k1) fetch(kb);
    for (int i = tid; i < a.NB * 32; i += 256) {
        const int b = i >> 5, c = i & 31;
        float v = 0.f;
        if (c < ncol) v = raw_bias(a.table[(int64_t)b * a.H + h0 + c], a.inv_scale);
        sb[i] = v;
    }
    bf16x8_t qf[KS];
    {
        const bf16_t* qp = a.Q + (int64_t)s * a.ldq + (int64_t)(h0 + (col ? r : 0)) * D + 8 * hh;
#pragma unroll
        for (int t = 0; t < KS; ++t) { qf[t] = ld_frag(qp + 16 * t); if (!col) qf[t] = zero_frag(); }
    }
    const int32_t* map = a.plan + a.far;                                // map[d], d = key - pos in [-far, 0]
    auto row_of = [&](int d) { const int b = map[d]; return b < 0 ? 0 : (b < a.NB ? b : a.NB - 1); };
    f32x16_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = splat16(0.f);
    float m = -INFINITY, l = 0.f;
    __syncthreads();
    const float cleft = sb[row_of(-a.far) * 32 + r];
    for (; kb < k1; kb += 128) {
        const bool tail = kb + 32 > k1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int id = lane + 64 * i;
            const int which = id / (32 * ROWP), rem = id - which * 32 * ROWP;
            const int rr = rem / ROWP, c = rem - rr * ROWP;
            u32x4_t w = sv[i];
            if (tail && kb + rr >= k1) w = (u32x4_t){0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4_t*>(sK + which * TILE + rr * DP + 8 * c) = w;
        }
        const bool near = kb + 31 - pos > -a.far;
        f32x16_t sc = splat16(cleft);
        if (near) {
#pragma unroll
            for (int reg = 0; reg < 16; ++reg) {
                int d = kb + ACC_ROW(reg, hh) - pos;
                d = d > 0 ? 0 : (d < -a.far ? -a.far : d);
                sc[reg] = sb[row_of(d) * 32 + r];
            }
        }
        if (kb + 128 < k1) fetch(kb + 128);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // the wave's own LDS tile: its instructions stay in order
#pragma unroll
        for (int t = 0; t < KS; ++t) sc = MFMA32(nat_frag<DP>(sK, r, hh, t), qf[t], sc);
        float x[16];
        float mr = -INFINITY;
#pragma unroll
        for (int reg = 0; reg < 16; ++reg) {
            x[reg] = tail && kb + ACC_ROW(reg, hh) >= k1 ? -INFINITY : sc[reg];
            mr = fmaxf(mr, x[reg]);
        }
        mr = half_max(mr);
        const float mx = fmaxf(m, mr * a.scale2);
        const float nm = mx == -INFINITY ? 0.f : -mx;
        const float alpha = __builtin_amdgcn_exp2f(m + nm);
        m = mx;
        float ls = 0.f;
#pragma unroll
        for (int reg = 0; reg < 16; ++reg) {
            x[reg] = __builtin_amdgcn_exp2f(fmaf(x[reg], a.scale2, nm));
            ls += x[reg];
        }
        ls = half_sum(ls);
        l = l * alpha + ls;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int reg = 0; reg < 16; ++reg) o[dt][reg] *= alpha;
        }
        const bf16x8_t p0 = pack8(x), p1 = pack8(x + 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            o[dt] = MFMA32(tr_frag<DP>(sV, dt, 0, hh, r), p0, o[dt]);
            o[dt] = MFMA32(tr_frag<DP>(sV, dt, 1, hh, r), p1, o[dt]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    // ---- the four waves meet: statistics, then the scaled outputs, summed in one order
    __syncthreads();
    float* st = reinterpret_cast<float*>(smem);                         // [4][32] maxima, [4][32] sums, then per wave [D][33] outputs
    float* so = st + 256;
    static_assert(1024 + 4 * D * 33 * 4 <= 8 * TILE * 2, "the waves' tiles hold the statistics and the outputs");
    if (hh == 0) { st[32 * wave + r] = m; st[128 + 32 * wave + r] = l; }
    __syncthreads();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmax2(M, st[32 * w + r]);
    const float nM = M == -INFINITY ? 0.f : -M;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += st[128 + 32 * w + r] * __builtin_amdgcn_exp2f(st[32 * w + r] + nM);
    const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
    const float f = __builtin_amdgcn_exp2f(m + nM) * inv;
    if (col) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int reg = 0; reg < 16; ++reg) so[(wave * D + 32 * dt + ACC_ROW(reg, hh)) * 33 + r] = f == 0.f ? 0.f : o[dt][reg] * f;
    }
    if (wave == 0 && hh == 0 && col && a.nsplit > 1)
        a.pl[((int64_t)s * a.nsplit + sp) * a.H + h0 + r] = L == 0.f ? -INFINITY : M + __log2f(L);
    __syncthreads();
    for (int i = tid; i < ncol * D; i += 256) {
        const int c = i / D, d = i - c * D;
        const float v = ((so[d * 33 + c] + so[(D + d) * 33 + c]) + so[(2 * D + d) * 33 + c]) + so[(3 * D + d) * 33 + c];
        if (a.nsplit == 1) a.O[(int64_t)s * a.ldo + (int64_t)(h0 + c) * D + d] = f2bf(v);
        else a.po[(((int64_t)s * a.nsplit + sp) * a.H + h0 + c) * D + d] = v;
    }
}

// joins the parts of a sequence: O = sum_p 2^(lse_p - M) O_p / sum_p 2^(lse_p - M).  A block per (sequence, head): wave w takes parts w, w + 4, ..., eight
// loads in flight, and the four sums meet in order.
template <int D>
__global__ void __launch_bounds__(256) relattn_parts_kernel(DP_ a) {
    constexpr int N = (D + 63) / 64;
    __shared__ float so[4][D], sw[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = blockIdx.x / a.H, h = blockIdx.x - s * a.H;
    int len = a.lens[s];
    len = len < 0 ? 0 : (len > a.cap ? a.cap : len);
    const int np = len == 0 ? 1 : (len + a.chunk - 1) / a.chunk;
    const float* pl = a.pl + ((int64_t)s * a.nsplit) * a.H + h;
    const float* po = a.po + ((int64_t)s * a.nsplit * a.H + h) * D;
    float M = -INFINITY;
    for (int p = lane; p < np; p += 64) M = fmax2(M, pl[(int64_t)p * a.H]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmax2(M, __shfl_xor(M, o, 64));
    const float nM = M == -INFINITY ? 0.f : -M;
    float w = 0.f, acc[N] = {};
#pragma unroll 8
    for (int p = wave; p < np; p += 4) {
        const float e = __builtin_amdgcn_exp2f(pl[(int64_t)p * a.H] + nM);
        w += e;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float v = lane + 64 * i < D ? po[(int64_t)p * a.H * D + lane + 64 * i] : 0.f;
            acc[i] = fmaf(e, e == 0.f ? 0.f : v, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane + 64 * i < D) so[wave][lane + 64 * i] = acc[i];
    if (lane == 0) sw[wave] = w;
    __syncthreads();
    if ((int)threadIdx.x < D) {
        w = ((sw[0] + sw[1]) + sw[2]) + sw[3];
        const float v = ((so[0][threadIdx.x] + so[1][threadIdx.x]) + so[2][threadIdx.x]) + so[3][threadIdx.x];
        a.O[(int64_t)s * a.ldo + (int64_t)h * D + threadIdx.x] = f2bf(w == 0.f ? 0.f : v / w);
    }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int MAX_FAR = 2048, MAX_NB = 256;      // the widest bias arrays (155 KB with the tiles at head dim 128) fit the 160 KB of LDS

constexpr int64_t MAX_LD = 1 << 24;               // a tile's 64 rows are addressed with 32-bit byte offsets

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check_bias(const char* who, const float* table, const int32_t* plan, int NB, int far, int causal, float scale) {
    STG_CHECK(table && plan, -1, "%s: null table / plan", who);
    STG_CHECK(NB >= (causal ? 2 : 4) && NB <= MAX_NB && (causal || NB % 2 == 0), -2, "%s: %d buckets (2..%d, even and >= 4 without the causal rule)", who, NB, MAX_NB);
    STG_CHECK(far >= 1 && far <= MAX_FAR, -2, "%s: the last bucket starts at distance %d (1..%d)", who, far, MAX_FAR);
    STG_CHECK(scale > 0.f && scale < 1e10f && scale > 1e-10f, -2, "%s: scale %g (1e-10 .. 1e10)", who, scale);
    return 0;
}

int check_args(const char* who, const stg_relattn_args* a) {
    STG_CHECK(a != nullptr, -1, "%s: null arguments", who);
    STG_CHECK(a->S >= 0 && a->S < 65535 && a->Tq >= 0 && a->Tk >= 0 && a->Tq <= INT32_MAX - 1024 && a->Tk <= INT32_MAX - 1024, -2,
              "%s: S=%d (< 65535), Tq=%lld, Tk=%lld (< 2^31 - 1024)", who, a->S, (long long)a->Tq, (long long)a->Tk);
    STG_CHECK((a->Tq == 0 || (a->Q && a->O)) && (a->Tk == 0 || (a->K && a->V)) && a->cu_q && a->cu_k, -1, "%s: null tensor", who);
    STG_CHECK(a->D == 32 || a->D == 64 || a->D == 96 || a->D == 128, -2, "%s: head dim %d (32, 64, 96 or 128)", who, a->D);
    STG_CHECK(a->H > 0 && a->H <= 65535 && a->Hkv > 0 && a->H % a->Hkv == 0, -2, "%s: %d heads over %d key / value heads", who, a->H, a->Hkv);
    STG_CHECK(a->max_q >= 0 && a->max_k >= 0, -2, "%s: max_q=%d, max_k=%d", who, a->max_q, a->max_k);
    const int64_t hd = (int64_t)a->H * a->D, kd = (int64_t)a->Hkv * a->D;
    STG_CHECK(a->ldq >= hd && a->ldo >= hd && a->ldk >= kd && a->ldv >= kd && a->ldq % 8 == 0 && a->ldk % 8 == 0 && a->ldv % 8 == 0 && a->ldo % 8 == 0, -3,
              "%s: leading dimensions must be multiples of 8 and hold every head", who);
    STG_CHECK(a->ldq <= MAX_LD && a->ldk <= MAX_LD && a->ldv <= MAX_LD && a->ldo <= MAX_LD, -3, "%s: leading dimensions up to 2^24", who);
    STG_CHECK(!misaligned(a->Q) && !misaligned(a->K) && !misaligned(a->V) && !misaligned(a->O), -3, "%s: tensors must be 16-byte aligned", who);
    return check_bias(who, a->table, a->plan, a->num_buckets, a->far, a->causal, a->scale);
}

RP make_rp(const stg_relattn_args* a) {
    RP p{};
    p.Q = (const bf16_t*)a->Q; p.ldq = a->ldq;
    p.K = (const bf16_t*)a->K; p.ldk = a->ldk;
    p.V = (const bf16_t*)a->V; p.ldv = a->ldv;
    p.O = (bf16_t*)a->O; p.ldo = a->ldo;
    p.lse = a->lse;
    p.cu_q = a->cu_q; p.cu_k = a->cu_k; p.kmask = (const uint8_t*)a->key_mask;
    p.Tq = a->Tq; p.Tk = a->Tk; p.S = a->S; p.H = a->H; p.Hkv = a->Hkv; p.causal = a->causal != 0; p.zero_tail = a->zero_tail == TAIL_LSE ? TAIL_LSE : a->zero_tail != 0;
    p.table = a->table; p.plan = a->plan; p.NB = a->num_buckets; p.far = a->far;
    p.hsplit = 1;
    p.scale = a->scale; p.scale2 = a->scale * LOG2E; p.inv_scale = 1.0f / a->scale;
    return p;
}

int64_t lds_fwd(int D, const RP& p) { return (int64_t)4 * 64 * (D + 8) * 2 + bias_len(p.far, p.causal) * 4; }
int64_t lds_dkv(int D, const RP& p, bool table) {
    const int64_t alen = (bias_len(p.far, p.causal) + 3) & ~3;
    return (int64_t)2 * (2 * 64 * (D + 8) + STATS) * 2 + alen * 4 + (table ? 2 * alen * 4 + 4 * 32 * 33 * 4 + alen : 0);
}
int64_t lds_dec(int D, int NB) { return (int64_t)8 * 32 * (D + 8) * 2 + (int64_t)NB * 32 * 4; }

int64_t cover(int max_n, int64_t T, int rows) {
    int64_t n = max_n > 0 ? max_n : 1;
    n = n < T ? n : (T > 0 ? T : 1);
    return (n + rows - 1) / rows;
}
// Blocks per (sequence, head): one per 128-row tile of the longest sequence, but no more than 2^18 over all of them (a hundred rounds on
// the chip); beyond, a block strides over several tiles.  Many short sequences without a length hint would otherwise launch tiles for sequences
// as long as the whole batch (1000 of 14 .. 100 rows, 16 heads: 7 million empty blocks).
int grid_tiles(int max_n, int64_t T, int64_t heads) {
    const int64_t t = cover(max_n, T, 128), most = ((int64_t)1 << 18) / (heads > 0 ? heads : 1);
    return (int)(t <= most ? t : (most < 1 ? 1 : most));
}
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;     // of 256 threads: a launch's threads are counted in 32 bits

template <int D>
int launch_fwd(const RP& p0, int max_q, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto k = relattn_fwd_kernel<D, 4>;
    STG_CHECK(stg_reserve_lds(k, 160 * 1024, done), -5, "stg_relattn_fwd: cannot reserve LDS");
    RP p = p0;
    p.tiles = grid_tiles(max_q, p.Tq, (int64_t)p.S * p.H);
    const int64_t blocks = (int64_t)p.tiles * p.H * (p.S + (p.zero_tail ? 1 : 0));
    STG_CHECK(blocks <= MAX_BLOCKS, -2, "relattn: %d sequences of %d heads are more than 2^24 blocks", p.S, p.H);
    if (blocks == 0) return 0;
    k<<<dim3((unsigned)blocks), 256, lds_fwd(D, p), st>>>(p);
    STG_LAUNCH_CHECK();
    return 0;
}
template <int D, bool TAB>
int launch_dq(const RP& p0, int max_q, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto k = relattn_dq_kernel<D, 4, TAB>;
    STG_CHECK(stg_reserve_lds(k, 160 * 1024, done), -5, "stg_relattn_bwd: cannot reserve LDS");
    RP p = p0;
    p.tiles = grid_tiles(max_q, p.Tq, (int64_t)p.S * p.H);
    const int64_t blocks = (int64_t)p.tiles * p.H * (p.S + (p.zero_tail ? 1 : 0));
    STG_CHECK(blocks <= MAX_BLOCKS, -2, "relattn: %d sequences of %d heads are more than 2^24 blocks", p.S, p.H);
    if (blocks == 0) return 0;
    k<<<dim3((unsigned)blocks), 256, lds_fwd(D, p), st>>>(p);
    STG_LAUNCH_CHECK();
    return 0;
}
template <int D, bool TAB>
int launch_dkv(const RP& p0, int max_k, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto k = relattn_dkv_kernel<D, 4, TAB>;
    STG_CHECK(stg_reserve_lds(k, 160 * 1024, done), -5, "stg_relattn_bwd: cannot reserve LDS");
    RP p = p0;
    p.tiles = grid_tiles(max_k, p.Tk, (int64_t)p.S * p.Hkv);
    const int64_t blocks = (int64_t)p.tiles * p.Hkv * p.hsplit * (p.S + (p.zero_tail && p.hsplit == 1 ? 1 : 0));
    STG_CHECK(blocks <= MAX_BLOCKS, -2, "relattn: %d sequences of %d heads are more than 2^24 blocks", p.S, p.H);
    if (blocks > 0) {
        k<<<dim3((unsigned)blocks), 256, lds_dkv(D, p, TAB), st>>>(p);
        STG_LAUNCH_CHECK();
    }
    if (p.hsplit > 1) {
        const int64_t n = (p.Tk * (p.Hkv * D / 4) + 255) / 256;
        relattn_kvsum_kernel<<<dim3((unsigned)(n < 2048 ? n : 2048)), 256, 0, st>>>(p, p.Hkv * D);
        STG_LAUNCH_CHECK();
    }
    return 0;
}
template <int D>
int launch_decode(const DP_& p, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    auto k = relattn_decode_kernel<D>;
    STG_CHECK(stg_reserve_lds(k, 160 * 1024, done), -5, "stg_relattn_decode: cannot reserve LDS");
    const int ncg = (p.H / p.Hkv + 31) / 32;
    k<<<dim3(p.nsplit, p.Hkv * ncg, p.S), 256, lds_dec(D, p.NB), st>>>(p);
    STG_LAUNCH_CHECK();
    if (p.nsplit > 1) {
        relattn_parts_kernel<D><<<dim3((unsigned)(p.S * p.H)), 256, 0, st>>>(p);
        STG_LAUNCH_CHECK();
    }
    return 0;
}

#define BY_DIM(D_, CALL)                                             \
    switch (D_) {                                                    \
        case 32: { constexpr int DIM = 32; return CALL; }            \
        case 64: { constexpr int DIM = 64; return CALL; }            \
        case 96: { constexpr int DIM = 96; return CALL; }            \
        default: { constexpr int DIM = 128; return CALL; }           \
    }

int run_fwd(const RP& p, int D, int max_q, hipStream_t st) {
    BY_DIM(D, (launch_fwd<DIM>(p, max_q, st)));
}
int run_dq(const RP& p, int D, int max_q, hipStream_t st) {
    if (p.part) BY_DIM(D, (launch_dq<DIM, true>(p, max_q, st)));
    BY_DIM(D, (launch_dq<DIM, false>(p, max_q, st)));
}
int run_dkv(const RP& p, int D, int max_k, hipStream_t st) {
    if (p.part) BY_DIM(D, (launch_dkv<DIM, true>(p, max_k, st)));
    BY_DIM(D, (launch_dkv<DIM, false>(p, max_k, st)));
}
int run_decode(const DP_& p, int D, hipStream_t st) { BY_DIM(D, (launch_decode<DIM>(p, st))); }

// Keys per block of the single-token form: about 1024 blocks at full length (two rounds of two per compute unit; 64 sequences of 1 .. 4096 tokens:
// 132 us against 145 / 199 us for blocks of 1024 / 512 keys), at least 128 keys (a 32-key tile for each of the four waves), at most 2048.
int decode_chunk(int S, int Hkv, int rep, int cap) {
    const int64_t groups = (int64_t)S * Hkv * ((rep + 31) / 32);
    const int64_t total = groups * cap;
    int64_t c = (total / 1024 + 127) / 128 * 128;
    c = c < 128 ? 128 : (c > 2048 ? 2048 : c);
    while ((cap + c - 1) / c > 4096) c *= 2;
    return (int)c;
}

}  // namespace

extern "C" int stg_relattn_fwd(const stg_relattn_args* a, void* stream) {
    const int rc = check_args("stg_relattn_fwd", a);
    if (rc) return rc;
    if (a->Tq == 0) return 0;
    return run_fwd(make_rp(a), a->D, a->max_q, (hipStream_t)stream);
}

// Blocks that share the query heads of a key / value head in the dK / dV kernel: as many as bring the launch to 1024 blocks (512 where heads are wide and blocks
// alike), by the rows alone, so that a length hint changes no bit.  Under the causal rule few blocks leave the longest walks for the end: 4 x 4096,
// 16 / 2 heads of 64 972 -> 560 us for the backward without the table, of 128 1728 -> 1212 us; the parts cost 8 bytes per element and block (29 us
// of 1.2 ms on 8112 rows of 8 x 128 in two parts).
static int head_split(const stg_relattn_args* a) {
    const int rep = a->H / a->Hkv;
    const int64_t blocks = (a->Tk / 128 + a->S) * a->Hkv, want = a->causal || a->D <= 64 ? 1024 : 512;
    int n = 1;
    while (n < rep && (rep % n != 0 || blocks * n < want)) ++n;
    return n;
}
static int64_t split_floats(const stg_relattn_args* a) {
    const int n = head_split(a);
    return n > 1 ? (int64_t)n * 2 * a->Tk * a->Hkv * a->D : 0;
}
// rows of the table's partial gradients: one per block of the dQ and of the dK / dV kernel (and head)
static int64_t behind_rows(const stg_relattn_args* a) { return a->Tq > 0 ? (int64_t)grid_tiles(a->max_q, a->Tq, (int64_t)a->S * a->H) * a->S : 0; }
static int64_t seen_words(const stg_relattn_args* a) { return behind_rows(a) * a->H * 4; }
static int64_t band_rows(const stg_relattn_args* a) { return a->Tq > 0 && a->Tk > 0 ? (int64_t)grid_tiles(a->max_k, a->Tk, (int64_t)a->S * a->Hkv) * a->S : 0; }

extern "C" int64_t stg_relattn_bwd_ws_floats(const stg_relattn_args* a, int want_table) {
    if (a == nullptr || a->S < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv != 0 || a->D <= 0 || a->Tq < 0 || a->Tk < 0 || a->num_buckets <= 0 || a->far <= 0) return -1;
    int64_t n = (int64_t)2 * a->H * a->Tq + seen_words(a) + split_floats(a);
    if (want_table) n += a->H * (behind_rows(a) * 2 + band_rows(a) * a->num_buckets);
    return n > 0 ? n : 1;
}

extern "C" int stg_relattn_bwd(const stg_relattn_args* a, const void* dO, int64_t lddo, void* dQ, int64_t lddq, void* dK, int64_t lddk, void* dV,
                               int64_t lddv, float* dtable, float* ws, int64_t ws_floats, void* stream) {
    const int rc = check_args("stg_relattn_bwd", a);
    if (rc) return rc;
    const int64_t hd = (int64_t)a->H * a->D, kd = (int64_t)a->Hkv * a->D;
    STG_CHECK((a->Tq == 0 || (dO && dQ && a->lse)) && (a->Tk == 0 || (dK && dV)) && ws, -1, "stg_relattn_bwd: null tensor");
    STG_CHECK(lddo <= MAX_LD, -3, "stg_relattn_bwd: leading dimensions up to 2^24");
    STG_CHECK(lddo >= hd && lddq >= hd && lddk >= kd && lddv >= kd && lddo % 8 == 0 && lddq % 8 == 0 && lddk % 8 == 0 && lddv % 8 == 0, -3,
              "stg_relattn_bwd: leading dimensions must be multiples of 8 and hold every head");
    STG_CHECK(!misaligned(dO) && !misaligned(dQ) && !misaligned(dK) && !misaligned(dV) && !misaligned(ws), -3, "stg_relattn_bwd: tensors must be 16-byte aligned");
    STG_CHECK(ws_floats >= stg_relattn_bwd_ws_floats(a, dtable != nullptr), -4, "stg_relattn_bwd: workspace of %lld floats is too small", (long long)ws_floats);
    hipStream_t st = (hipStream_t)stream;
    RP p = make_rp(a);
    p.dO = (const bf16_t*)dO; p.lddo = lddo; p.dQ = (bf16_t*)dQ; p.lddq = lddq;
    p.dK = (bf16_t*)dK; p.lddk = lddk; p.dV = (bf16_t*)dV; p.lddv = lddv;
    p.zero_tail = p.zero_tail == 1;
    p.hsplit = head_split(a);
    p.pk = ws;
    p.delta = ws + split_floats(a);
    p.fix = p.delta + (int64_t)a->H * a->Tq;
    p.seen = reinterpret_cast<uint32_t*>(p.fix + (int64_t)a->H * a->Tq);
    p.qtiles = a->Tq > 0 ? grid_tiles(a->max_q, a->Tq, (int64_t)a->S * a->H) : 0;
    float* behind = p.fix + (int64_t)a->H * a->Tq + seen_words(a);
    float* band = behind + behind_rows(a) * a->H * 2;
    p.part = dtable ? behind : nullptr;
    if (a->Tq > 0) { const int e = run_dq(p, a->D, a->max_q, st); if (e) return e; }
    if (dtable) p.part = band_rows(a) > 0 ? band : nullptr;
    if (a->Tk > 0) { const int e = run_dkv(p, a->D, a->max_k, st); if (e) return e; }
    if (dtable) {
        relattn_dtable_kernel<<<dim3(a->H, a->num_buckets), 256, 0, st>>>(band, (int)band_rows(a), behind, (int)behind_rows(a), dtable, a->H, a->num_buckets, a->causal != 0);
        STG_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int64_t stg_relattn_decode_ws_floats(int S, int cap, int H, int Hkv, int D) {
    if (S <= 0 || cap <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0) return 0;
    const int c = decode_chunk(S, Hkv, H / Hkv, cap);
    const int64_t ns = (cap + c - 1) / c;
    return ns > 1 ? (int64_t)S * ns * H * (D + 1) : 0;
}

extern "C" int stg_relattn_decode(const stg_relattn_decode_args* a, float* ws, int64_t ws_floats, void* stream) {
    STG_CHECK(a != nullptr, -1, "stg_relattn_decode: null arguments");
    STG_CHECK(a->S >= 0 && a->S <= 65535 && a->cap >= 0 && a->cap <= INT32_MAX - 1024, -2, "stg_relattn_decode: S=%d (<= 65535), cap=%d", a->S, a->cap);
    STG_CHECK(a->D == 32 || a->D == 64 || a->D == 96 || a->D == 128, -2, "stg_relattn_decode: head dim %d (32, 64, 96 or 128)", a->D);
    STG_CHECK(a->H > 0 && a->H <= 32768 && (int64_t)a->H * a->S <= MAX_BLOCKS && a->Hkv > 0 && a->H % a->Hkv == 0, -2, "stg_relattn_decode: %d heads over %d key / value heads", a->H, a->Hkv);
    STG_CHECK(a->Q && a->O && a->lens && (a->cap == 0 || (a->K && a->V)), -1, "stg_relattn_decode: null tensor");
    const int64_t hd = (int64_t)a->H * a->D, kd = (int64_t)a->Hkv * a->D;
    STG_CHECK(a->ldq >= hd && a->ldo >= hd && a->ldk >= kd && a->ldv >= kd && a->ldq % 8 == 0 && a->ldk % 8 == 0 && a->ldv % 8 == 0 && a->bsk % 8 == 0 &&
              a->bsv % 8 == 0 && a->bsk >= 0 && a->bsv >= 0, -3, "stg_relattn_decode: strides must be multiples of 8 and hold every head");
    STG_CHECK(!misaligned(a->Q) && !misaligned(a->K) && !misaligned(a->V), -3, "stg_relattn_decode: tensors must be 16-byte aligned");
    const int rc = check_bias("stg_relattn_decode", a->table, a->plan, a->num_buckets, a->far, a->causal, a->scale);
    if (rc) return rc;
    if (a->S == 0) return 0;
    DP_ p{};
    p.Q = (const bf16_t*)a->Q; p.ldq = a->ldq;
    p.K = (const bf16_t*)a->K; p.ldk = a->ldk; p.bsk = a->bsk;
    p.V = (const bf16_t*)a->V; p.ldv = a->ldv; p.bsv = a->bsv;
    p.O = (bf16_t*)a->O; p.ldo = a->ldo;
    p.lens = a->lens; p.S = a->S; p.cap = a->cap; p.H = a->H; p.Hkv = a->Hkv;
    p.table = a->table; p.plan = a->plan; p.NB = a->num_buckets; p.far = a->far;
    p.scale2 = a->scale * LOG2E; p.inv_scale = 1.0f / a->scale;
    const int cap1 = a->cap > 0 ? a->cap : 1;
    p.chunk = decode_chunk(a->S, a->Hkv, a->H / a->Hkv, cap1);
    p.nsplit = (cap1 + p.chunk - 1) / p.chunk;
    const int64_t need = stg_relattn_decode_ws_floats(a->S, a->cap, a->H, a->Hkv, a->D);
    STG_CHECK(need == 0 || (ws != nullptr && ws_floats >= need), -4, "stg_relattn_decode: workspace of %lld floats is too small", (long long)ws_floats);
    p.po = ws;
    p.pl = ws ? ws + (int64_t)a->S * p.nsplit * a->H * a->D : nullptr;
    return run_decode(p, a->D, (hipStream_t)stream);
}
