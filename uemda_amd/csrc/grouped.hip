// Products of feature rows with the weight of the group each row belongs to, the rows sorted by group and the groups' sizes known on the
// device only (offsets[g] .. offsets[g + 1] are the rows of group g):
//   forward          y[r]  = W_g x[r] + b_g         x [T][K], W [G][N][K], y [T][N]
//   data gradient    dx[r] = W_g^T dy[r]
//   weight gradient  dW_g  = sum over the group's rows of dy[r] x[r]^T,   db_g = sum of dy[r]
// Rows in front of offsets[0] and behind offsets[G] belong to no group: their y and dx are zeros and they enter no gradient.
//
// Matrix-bound (2 T K N flops each) once a group has some hundred rows, bound by reading W below.  One kernel serves the three: an
// operand tile travels global -> LDS by 16-byte LDS-DMA, 64 bytes of the reduction index per tile row a stage, four stages;
// where the reduction index is the SLOW one in memory (W in the data gradient, both operands of the weight gradient) the image is kept as
// it sits in memory and read transposed: bf16 by ds_read_b64_tr_b16, fp32 by consecutive ds_read_b32.  Both kinds are XOR-swizzled in
// 16-byte chunks on the source address so that a read covers all banks.  Buffer descriptors that end with the group's last row (and
// offsets beyond them for columns past the end) supply the zeros of every ragged edge: no row of another group is ever read.
// Products are exact in the fp32 accumulators (bf16) or fp32 MFMA (fp32); bf16 results are rounded once.
//
// Nothing is read on the host: a block finds its tile by scanning the offsets (a wave's prefix sums, ~0.5 us for up to 62 groups), the grid
// is the most tiles T rows in G groups can make.  Offsets are clamped to [0, T] and to the largest one in front of them, so that any
// contents give disjoint groups inside the tensors.
#include "common.h"

namespace {

typedef unsigned short bf16_t;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) unsigned int* lds_u32p;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4p;

}  // namespace
// buffer_load_dwordx4 ... lds: per-lane global offset, LDS destination = wave-uniform base (M0) + lane * 16
extern "C" __device__ void uem_raw_buffer_load_lds(i32x4 rsrc, lds_u32p lds, int size, int voffset, int soffset, int offset,
                                                   int aux) __asm("llvm.amdgcn.raw.buffer.load.lds");
namespace {

constexpr unsigned GG_OOB = 0xFFFFFFF0u;          // beyond every descriptor: the load returns zeros
constexpr int FWD = 0, DGRAD = 1, WGRAD = 2;

struct GgP {
    const char* a; const char* b;                 // FWD x, W | DGRAD dy, W | WGRAD dy, x
    char* out;
    const void* bias;                             // FWD only, may be null
    float* part;                                  // WGRAD: partial sums of groups of several row chunks
    const void* offsets;
    int64_t lda, ldb;                             // bytes of a row of a / of b
    int T, G, K, N, chunk;                        // K: columns of x (out of W's rows), N: columns of y;  chunk: rows of a WGRAD item
    int64_t ldo;                                  // elements of an output row
    bool off64, bias16, out16, vec;               // 64-bit offsets; bias / output in bf16; output rows take 16-byte stores
};

__device__ __forceinline__ i32x4 rsrc(const char* p, unsigned bytes) {
    const unsigned long long a = (unsigned long long)p;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffu));
    r[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffffu));
    r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
    r[3] = 0x00020000;
    return r;
}

// ---- which rows ---------------------------------------------------------------------------------------------------------------------
// Segments of the rows: ALL: 0 = the rows in front of the first group, 1 .. G the groups, G + 1 the rows behind the last; !ALL: the groups.
struct Seg {
    int seg, row0, rows, tile;                    // segment, its first row and length, tile within it
    int total, before, nslots, slot;              // tiles in all; tiles before this segment; partial-sum slots in all, this segment's first
};
__device__ __forceinline__ int gg_offset(const GgP& p, int i) {
    int64_t o = p.off64 ? ((const int64_t*)p.offsets)[i] : (int64_t)((const int*)p.offsets)[i];
    o = o < 0 ? 0 : o;
    return (int)(o > p.T ? p.T : o);
}
__device__ __forceinline__ int scan_add(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o, 64); if (lane >= o) v += u; }
    return v;
}
__device__ __forceinline__ int scan_max(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o, 64); if (lane >= o) v = u > v ? u : v; }
    return v;
}
// Tiles of `bm` rows (!ALL: an empty group still has one, which writes its zeros).  Pass 0 counts them; `want` (a function of the count:
// which tile this block takes, < 0 for none) is then found in pass 1 -- the same pass where all segments fit one wave.  Slots are counted
// over groups of several tiles only.
template <bool ALL, typename Want>
__device__ __forceinline__ bool find_tile(const GgP& p, int bm, Want want, Seg& s) {
    const int lane = threadIdx.x & 63, nseg = ALL ? p.G + 2 : p.G, chunks = (nseg + 63) >> 6;
    int target = -1;
    s.total = s.nslots = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int edge = ALL ? 0 : gg_offset(p, 0), tiles = 0, slots = 0;
        for (int c = 0; c < chunks; ++c) {
            const int v = c * 64 + lane;
            int end = v < nseg ? (ALL ? (v <= p.G ? gg_offset(p, v) : p.T) : gg_offset(p, v + 1)) : 0;
            end = scan_max(end > edge ? end : edge, lane);
            const int up = __shfl_up(end, 1, 64), begin = lane == 0 ? edge : up;
            const int len = end - begin;
            int nt = v < nseg ? (len + bm - 1) / bm : 0;
            if (!ALL && v < nseg && nt == 0) nt = 1;
            const int sum = scan_add(nt, lane) + tiles, ns = ALL ? 0 : scan_add(nt > 1 ? nt : 0, lane) + slots;
            if (pass == 1 || chunks == 1) {
                if (chunks == 1) {
                    s.total = __shfl(sum, 63, 64);
                    s.nslots = ALL ? 0 : __shfl(ns, 63, 64);
                    target = want(s.total);
                    if (target < 0) return false;
                }
                const unsigned long long hit = __ballot(sum > target);
                if (hit != 0) {
                    const int l = __builtin_ctzll(hit);
                    s.seg = c * 64 + l;
                    s.before = __shfl(sum - nt, l, 64);
                    s.tile = target - s.before;
                    s.row0 = __shfl(begin, l, 64);
                    s.rows = __shfl(len, l, 64);
                    s.slot = ALL ? 0 : __shfl(ns - (nt > 1 ? nt : 0), l, 64);
                    return true;
                }
            }
            edge = __shfl(end, 63, 64);
            tiles = __shfl(sum, 63, 64);
            slots = ALL ? 0 : __shfl(ns, 63, 64);
        }
        if (pass == 0) {
            s.total = tiles;
            s.nslots = slots;
            target = want(s.total);
            if (target < 0) return false;
        }
    }
    return false;
}
// Blocks go to the eight XCDs in turn: each gets one contiguous run of the n items, neighbours share their operand tiles in its L2.
__device__ __forceinline__ int xcd_item(int n) {
    const int x = blockIdx.x & 7, i = blockIdx.x >> 3, per = n >> 3, rem = n & 7;
    return i < per + (x < rem ? 1 : 0) ? x * per + (x < rem ? x : rem) + i : -1;
}

// ---- operand images -------------------------------------------------------------------------------------------------------------------
// A stage holds 64 bytes of the reduction index (32 bf16, 16 fp32) of every tile row.
// KC (reduction index contiguous in memory): [R rows][64 bytes], chunk c of row r in slot c ^ ((r >> 2) & 3): the 16 rows a quarter-wave
// of ds_read_b128 touches fall on 16 different 16-byte slots of the 256-byte bank row.
// KS (reduction index slow): [64 / ES reduction rows][R columns]; bf16: chunk c of row r in slot c ^ ((r & 3) << 2): the four rows of a
// transposing read fall on the four quarters of the bank row.
template <int ES> __device__ __forceinline__ int ks_swz(int row) { return ES == 2 ? (row & 3) << 2 : 0; }

template <typename T, bool KS, int R, int NW>
struct Loader {
    static constexpr int ES = sizeof(T), PIECES = R / 16, IPW = PIECES / NW, ROWB = R * ES, LPR = ROWB / 16, RPP = 1024 / ROWB > 0 ? 1024 / ROWB : 1;
    static_assert(PIECES % NW == 0, "whole pieces a wave");
    unsigned off[IPW];
    int kc[IPW];                                  // KC: first reduction index of the lane's chunk
    // KC: `cols` is the reduction length, `bytes` a row's stride.  KS: the tile's first column and the columns there are
    __device__ __forceinline__ void init(int wave, int lane, int64_t bytes, int col0, int cols) {
#pragma unroll
        for (int j = 0; j < IPW; ++j) {
            const int q = j * NW + wave;
            if (!KS) {
                const int row = q * 16 + (lane >> 2), ch = (lane & 3) ^ ((row >> 2) & 3);
                off[j] = (unsigned)(row * bytes + ch * 16);
                kc[j] = ch * (16 / ES);
            } else {
                const int row = q * RPP + lane / LPR, ch = (lane % LPR) ^ ks_swz<ES>(row), col = col0 + ch * (16 / ES);
                off[j] = col < cols ? (unsigned)(row * bytes + (int64_t)col * ES) : GG_OOB;
                kc[j] = 0;
            }
        }
    }
    __device__ __forceinline__ void issue(const i32x4 rs, char* img, int wave, unsigned step_bytes, int k0, int klen) const {
#pragma unroll
        for (int j = 0; j < IPW; ++j) {
            const unsigned o = KS ? off[j] : (k0 + kc[j] < klen ? off[j] + step_bytes : GG_OOB);
            uem_raw_buffer_load_lds(rs, (lds_u32p)(img + (j * NW + wave) * 1024), 16, (int)o, 0, 0, 0);
        }
    }
};

// the operand of 32 tile rows (or columns) at r0 for reduction step ks of the stage: bf16 8 consecutive reduction indices a lane, fp32 four
template <typename T, bool KS, int R> struct Frag;
template <int R> struct Frag<bf16_t, false, R> {
    bf16x8 v;
    __device__ __forceinline__ void load(const char* img, int r0, int ks, int lane) {
        const int r = r0 + (lane & 31), ch = (2 * ks + (lane >> 5)) ^ ((r >> 2) & 3);
        v = *reinterpret_cast<const bf16x8*>(img + r * 64 + ch * 16);
    }
};
template <int R> struct Frag<bf16_t, true, R> {
    bf16x8 v;
    __device__ __forceinline__ void load(const char* img, int r0, int ks, int lane) {
        const int q = (lane & 15) >> 2, pp = lane & 3, g16 = (lane >> 4) & 1;
        const int row = ks * 16 + 8 * (lane >> 5) + q, ch = (r0 >> 3) + 2 * g16 + (pp >> 1);
        const char* const a0 = img + row * (R * 2) + ((ch ^ ks_swz<2>(row)) << 4) + ((pp & 1) << 3);
        const char* const a1 = img + (row + 4) * (R * 2) + ((ch ^ ks_swz<2>(row + 4)) << 4) + ((pp & 1) << 3);
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4p)(a0));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4p)(a1));
        v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};
template <int R> struct Frag<float, false, R> {
    f32x4 v;
    __device__ __forceinline__ void load(const char* img, int r0, int ks, int lane) {
        const int r = r0 + (lane & 31), ch = (2 * ks + (lane >> 5)) ^ ((r >> 2) & 3);
        v = *reinterpret_cast<const f32x4*>(img + r * 64 + ch * 16);
    }
};
template <int R> struct Frag<float, true, R> {
    f32x4 v;
    __device__ __forceinline__ void load(const char* img, int r0, int ks, int lane) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(img + (ks * 8 + 4 * (lane >> 5) + e) * (R * 4) + (r0 + (lane & 31)) * 4);
    }
};
template <typename FA, typename FB> __device__ __forceinline__ void mma(const FA& a, const FB& b, f32x16& c, bf16_t) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
template <typename FA, typename FB> __device__ __forceinline__ void mma(const FA& a, const FB& b, f32x16& c, float) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}

__device__ __forceinline__ unsigned bf_bits(float f) { return (unsigned)__builtin_bit_cast(unsigned short, (__bf16)f); }

// own LDS-DMA pieces but the last N, and own LDS accesses, complete; then everybody's
template <int N> __device__ __forceinline__ void gg_wait() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void gg_barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Four stages: the pieces of stage t + 3 leave while stage t is computed on, a wait is for pieces that left two stages ago.
// PP (eight waves, one block a CU): the two waves of a SIMD take turns -- while one feeds the matrix cores from registers, the other reads
// its next fragments and sends pieces off, a barrier between the turns.  With the waves in step both wait for LDS at the same time.
template <typename T, int FORM, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void grouped_kernel(const GgP p) {
    constexpr int ES = sizeof(T), NW = WGM * WGN, MT = BM / WGM / 32, NT = BN / WGN / 32, BK = 64 / ES, SB = (BM + BN) * 64, NST = 4;
    constexpr bool PP = NW == 8;
    constexpr bool AKS = FORM == WGRAD, BKS = FORM != FWD;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- this block's tile
    const int width = FORM == FWD ? p.N : p.K;                                 // output columns
    const int ct = (width + BN - 1) / BN, rt = FORM == WGRAD ? (p.N + BM - 1) / BM : 1;
    Seg s;
    int item = -1;
    if (!find_tile<FORM != WGRAD>(p, FORM == WGRAD ? p.chunk : BM, [&](int total) {
            item = xcd_item(total * ct * rt);
            return item < 0 ? -1 : item / (ct * rt);
        }, s)) return;
    s.seg = __builtin_amdgcn_readfirstlane(s.seg);
    s.row0 = __builtin_amdgcn_readfirstlane(s.row0);
    s.rows = __builtin_amdgcn_readfirstlane(s.rows);
    s.tile = __builtin_amdgcn_readfirstlane(s.tile);
    const int within = item % (ct * rt), c0 = (within % ct) * BN, n0 = (within / ct) * BM;      // n0: first row of W (WGRAD)
    const bool none = FORM != WGRAD && (s.seg == 0 || s.seg == p.G + 1);
    const int g = FORM == WGRAD ? s.seg : s.seg - 1;
    const int r0 = s.row0 + s.tile * (FORM == WGRAD ? p.chunk : BM);           // first feature row of the tile / of the chunk
    int rows = s.rows - s.tile * (FORM == WGRAD ? p.chunk : BM);               // feature rows of it
    rows = rows < 0 ? 0 : rows < (FORM == WGRAD ? p.chunk : BM) ? rows : (FORM == WGRAD ? p.chunk : BM);

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int wm = (wave / WGN) * (MT * 32), wn = (wave % WGN) * (NT * 32);

    // ---- operands: where they begin, how far they reach, how long the reduction is
    const int red = FORM == FWD ? p.K : FORM == DGRAD ? p.N : rows;            // reduction length
    const int steps = none ? 0 : (red + BK - 1) / BK;
    Loader<T, AKS, BM, NW> la;
    Loader<T, BKS, BN, NW> lb;
    la.init(wave, lane, p.lda, n0, p.N);
    lb.init(wave, lane, p.ldb, c0, p.K);
    const char* pa = p.a + (int64_t)r0 * p.lda;
    const char* pb = FORM == FWD ? p.b + ((int64_t)g * p.N + c0) * p.ldb : FORM == DGRAD ? p.b + (int64_t)g * p.N * p.ldb : p.b + (int64_t)r0 * p.ldb;
    // bytes of a row, up to the 16-byte boundary behind its last element (zeros there)
    const unsigned acols = (unsigned)((FORM == FWD ? p.K : p.N) * ES + 15) & ~15u, bcols = (unsigned)(p.K * ES + 15) & ~15u;
    int arem = rows, brem = FORM == FWD ? (p.N - c0 < BN ? p.N - c0 : BN) : FORM == DGRAD ? p.N : rows;    // rows left of a and b
    int q = 0;                                                                 // the next step to issue

    constexpr int IPW = Loader<T, AKS, BM, NW>::IPW + Loader<T, BKS, BN, NW>::IPW;
    auto issue = [&](char* __restrict__ fill) {                                // steps past the end fetch zeros: the counts of the waits hold
        const int na = AKS && arem > BK ? BK : arem, nb = BKS && brem > BK ? BK : brem;
        const i32x4 ra = rsrc(pa, na > 0 ? (unsigned)((na - 1) * p.lda) + acols : 0u), rb = rsrc(pb, nb > 0 ? (unsigned)((nb - 1) * p.ldb) + bcols : 0u);
        la.issue(ra, fill, wave, (unsigned)q * 64u, q * BK, red);
        lb.issue(rb, fill + BM * 64, wave, (unsigned)q * 64u, q * BK, red);
        if (AKS) { pa += BK * p.lda; arem -= BK; }
        if (BKS) { pb += BK * p.ldb; brem -= BK; }
        ++q;
    };
    Frag<T, AKS, BM> fa[2][MT];
    Frag<T, BKS, BN> fb[2][NT];
    // one function with the stage being refilled and the stage being read as __restrict__ pointers: that is what tells the compiler that
    // the reads do not depend on the LDS-DMA in flight (it would wait for all of it in front of the first read)
    auto stage = [&](char* __restrict__ fill, const char* __restrict__ use) {
        auto fetch = [&](const int ks) {
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[ks][i].load(use, wm + i * 32, ks, lane);
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[ks][j].load(use + BM * 64, wn + j * 32, ks, lane);
        };
        auto multiply = [&](const int ks) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) mma(fa[ks][i], fb[ks][j], acc[i][j], T{});
        };
        if (PP) {
            fetch(0);
            fetch(1);
            issue(fill);
            gg_wait<2 * IPW>();
            gg_barrier();
            __builtin_amdgcn_s_setprio(1);
            multiply(0);
            multiply(1);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            gg_barrier();
        } else {
            gg_wait<2 * IPW>();
            gg_barrier();
            issue(fill);
            fetch(0);
            fetch(1);
            multiply(0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(1);
        }
    };
    if (steps > 0) {
#pragma unroll
        for (int t = 0; t < NST - 1; ++t) issue(smem + t * SB);
        if (PP) {
            gg_wait<2 * IPW>();
            gg_barrier();
            if (wave >= NW / 2) gg_barrier();
        }
        for (int t = 0; t < steps; ++t) stage(smem + ((t + NST - 1) % NST) * SB, smem + (t % NST) * SB);
        if (PP && wave < NW / 2) gg_barrier();
    }

    // ---- results: MFMA column = lane & 31, row = (r & 3) + 8 (r >> 2) + 4 (lane >> 5)
    const int fr = lane & 31, fh = lane >> 5;
    float bias[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        bias[j] = 0.f;
        const int c = c0 + wn + j * 32 + fr;
        if (FORM == FWD && p.bias != nullptr && !none && c < p.N) {
            const int64_t i = (int64_t)g * p.N + c;
            bias[j] = p.bias16 ? __uint_as_float((uint32_t)((const bf16_t*)p.bias)[i] << 16) : ((const float*)p.bias)[i];
        }
    }
    // a chunk of a group with several goes to its partial-sum slot, in fp32
    const bool partial = FORM == WGRAD && s.rows > p.chunk;
    const int orow0 = FORM == WGRAD ? n0 : r0;                                 // first output row of the tile
    const int orows = FORM == WGRAD ? p.N - n0 : rows;
    const int64_t base = FORM == WGRAD ? (partial ? (int64_t)(s.slot + s.tile) : (int64_t)g) * p.N * p.K : 0;
    const int64_t ldo = FORM == WGRAD ? p.K : p.ldo;
    const bool o16 = partial ? false : p.out16;
    char* const out = partial ? (char*)p.part : p.out;
    const bool vec = partial ? (p.K & 3) == 0 : p.vec;
    gg_wait<0>();                                                              // everybody has read the last stage and nothing is on its way:
    gg_barrier();                                                              // the stages' memory takes the results
    constexpr int STG = NST * SB / NW;
    static_assert(STG >= 32 * NT * 32 * 4, "a wave's 32 result rows");
    char* const mine = smem + wave * STG;
    auto leave = [&](auto out_t) {
        using O = decltype(out_t);
        constexpr int ROWB = NT * 32 * sizeof(O), PER = 16 / sizeof(O), LPR = ROWB / 16;
        char* const put = mine + (4 * fh) * ROWB + fr * sizeof(O);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float v = acc[i][j][r] + bias[j];
                    O* const d = reinterpret_cast<O*>(put + ((r & 3) + 8 * (r >> 2)) * ROWB + j * 32 * sizeof(O));
                    if (sizeof(O) == 2) *d = (O)bf_bits(v);
                    else *d = (O)v;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // the wave's own rows, written by all its lanes
            const int left = orows - (wm + i * 32), rr = left < 32 ? left : 32;
            O* const dst = reinterpret_cast<O*>(out) + base + (int64_t)(orow0 + wm + i * 32) * ldo + c0 + wn;
            if (vec) {
#pragma unroll
                for (int t = 0; t < 32; t += 64 / LPR) {
                    const int row = t + lane / LPR, col = (lane % LPR) * PER;
                    if (row < rr && c0 + wn + col < width)
                        *reinterpret_cast<uint4*>(dst + row * ldo + col) = *reinterpret_cast<const uint4*>(mine + row * ROWB + (lane % LPR) * 16);
                }
            } else {
                for (int t = lane; t < 32 * NT * 32; t += 64) {
                    const int row = t / (NT * 32), col = t % (NT * 32);
                    if (row < rr && c0 + wn + col < width) dst[row * ldo + col] = reinterpret_cast<const O*>(mine)[t];
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (o16) leave(bf16_t{});
    else leave(float{});
}

// dW of the groups of several chunks = their partial sums, added in row order.  blockIdx.y: group
__global__ __launch_bounds__(256) void grouped_join_kernel(const GgP p) {
    const int g = blockIdx.y;
    int edge = gg_offset(p, 0), slots = 0, len = 0, first = 0;
    const int lane = threadIdx.x & 63;
    for (int c = 0; c * 64 <= g; ++c) {
        const int v = c * 64 + lane;
        int end = v < p.G ? gg_offset(p, v + 1) : 0;
        end = scan_max(end > edge ? end : edge, lane);
        const int up = __shfl_up(end, 1, 64), l = end - (lane == 0 ? edge : up);
        const int nt = v < p.G ? (l + p.chunk - 1) / p.chunk : 0, m = nt > 1 ? nt : 0;
        const int ns = scan_add(m, lane) + slots;
        if (g < c * 64 + 64) { len = __shfl(l, g & 63, 64); first = __shfl(ns - m, g & 63, 64); }
        edge = __shfl(end, 63, 64);
        slots = __shfl(ns, 63, 64);
    }
    if (len <= p.chunk) return;
    const int n = (len + p.chunk - 1) / p.chunk;
    const int64_t size = (int64_t)p.N * p.K;
    const float* const part = p.part + first * size;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int c = 0; c < n; ++c) v += part[c * size + i];
        if (p.out16) reinterpret_cast<bf16_t*>(p.out)[g * size + i] = (bf16_t)bf_bits(v);
        else reinterpret_cast<float*>(p.out)[g * size + i] = v;
    }
}

// db: column sums of dy per group.  Item: GG_BIAS_ROWS rows x 64 columns, four waves down the rows -> part[item's chunk][N]
constexpr int GG_BIAS_ROWS = 512;
template <typename T>
__global__ __launch_bounds__(256) void grouped_colsum_kernel(GgP p) {
    __shared__ float join[4][64];
    const int ct = (p.N + 63) / 64;
    Seg s;
    int item = -1;
    if (!find_tile<false>(p, GG_BIAS_ROWS, [&](int total) { item = (int)blockIdx.x < total * ct ? (int)blockIdx.x : -1; return item < 0 ? -1 : item / ct; }, s)) return;
    const int c = (item % ct) * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
    const int r0 = s.row0 + s.tile * GG_BIAS_ROWS, rows = min(GG_BIAS_ROWS, s.rows - s.tile * GG_BIAS_ROWS);
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < p.N) {
        const char* const src = p.a + (int64_t)r0 * p.lda + (int64_t)c * sizeof(T);
        auto at = [&](int r) { return sizeof(T) == 2 ? __uint_as_float((uint32_t)*(const bf16_t*)(src + r * p.lda) << 16) : *(const float*)(src + r * p.lda); };
        int r = w;
        for (; r + 12 < rows; r += 16)
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] += at(r + 4 * k);
        for (; r < rows; r += 4) a[0] += at(r);
    }
    join[w][threadIdx.x & 63] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (w == 0 && c < p.N) p.part[(int64_t)(s.before + s.tile) * p.N + c] = (join[0][threadIdx.x] + join[1][threadIdx.x]) + (join[2][threadIdx.x] + join[3][threadIdx.x]);
}
// db[g] = its chunks' sums in row order.  blockIdx.y: group
__global__ __launch_bounds__(256) void grouped_colsum_join_kernel(GgP p) {
    const int g = blockIdx.y, lane = threadIdx.x & 63, c = blockIdx.x * 256 + threadIdx.x;
    int edge = gg_offset(p, 0), tiles = 0, n = 0, first = 0;
    for (int k = 0; k * 64 <= g; ++k) {
        const int v = k * 64 + lane;
        int end = v < p.G ? gg_offset(p, v + 1) : 0;
        end = scan_max(end > edge ? end : edge, lane);
        const int up = __shfl_up(end, 1, 64), l = end - (lane == 0 ? edge : up);
        int nt = v < p.G ? (l + GG_BIAS_ROWS - 1) / GG_BIAS_ROWS : 0;
        if (v < p.G && nt == 0) nt = 1;
        const int sum = scan_add(nt, lane) + tiles;
        if (g < k * 64 + 64) { n = __shfl(nt, g & 63, 64); first = __shfl(sum - nt, g & 63, 64); }
        edge = __shfl(end, 63, 64);
        tiles = __shfl(sum, 63, 64);
    }
    if (c >= p.N) return;
    float v = 0.f;
    for (int k = 0; k < n; ++k) v += p.part[(int64_t)(first + k) * p.N + c];
    const int64_t i = (int64_t)g * p.N + c;
    if (p.out16) ((bf16_t*)p.out)[i] = (bf16_t)bf_bits(v);
    else ((float*)p.out)[i] = v;
}

// dst[r][0 .. ldd) = src[r][0 .. cols), zeros behind: rows that begin on 16-byte boundaries
template <typename T>
__global__ __launch_bounds__(256) void grouped_pad_kernel(const T* __restrict__ src, int64_t lds, T* __restrict__ dst, int ldd, int cols, int64_t rows) {
    const int64_t n = rows * ldd;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / ldd;
        const int c = (int)(i - r * ldd);
        dst[i] = c < cols ? src[r * lds + c] : (T)0;
    }
}

template <typename T, int FORM, int BM, int BN, int WGM, int WGN>
void go(const GgP& p, int64_t items, hipStream_t st) {
    constexpr int LDS = 4 * (BM + BN) * 64;
    auto k = grouped_kernel<T, FORM, BM, BN, WGM, WGN>;
    if (!uem_allow_lds((const void*)k, LDS)) return;
    k<<<(unsigned)items, 64 * WGM * WGN, LDS, st>>>(p);
}

// most row tiles that T rows in G groups make, with the rows in front and behind
int64_t most_tiles(int T, int G, int bm) { return T / bm + (int64_t)G + 2; }

// Tile of the forward and the data gradient.  256 x 256 moves the fewest operand bytes a flop; it needs enough tiles to fill the CUs and
// groups that fill it.  64 x 128 is for groups of a few rows, where the weight's bytes are what counts.
int tile_rows(int T, int G, int width) {
    const int64_t per = uem_cdiv(T, G);
    if (per >= 192 && (uem_cdiv(T, 256) + G / 2) * uem_cdiv(width, 256) >= 192) return 256;
    return per >= 80 ? 128 : 64;
}
// rows of a weight-gradient item: all of them where the groups' tiles fill the chip anyway, else so that it is filled
int wgrad_chunk(int T, int G, int N, int K, int bm) {
    const int64_t tiles = uem_cdiv(N, bm) * uem_cdiv(K, bm);
    int64_t c = uem_cdiv((int64_t)T * tiles, 256);
    c = uem_cdiv(c < 1024 ? 1024 : c, 64) * 64;
    return (int)(c > T ? (T < 64 ? 64 : uem_cdiv(T, 64) * 64) : c);
}
int wgrad_tile(int G, int N, int K) { return uem_cdiv(N, 256) * uem_cdiv(K, 256) * G >= 96 && N > 128 && K > 128 ? 256 : 128; }

template <typename T, int FORM>
int launch_rows(const GgP& p, const char* what, hipStream_t st) {
    const int width = FORM == FWD ? p.N : p.K, bm = tile_rows(p.T, p.G, width), bn = bm == 256 ? 256 : 128;
    const int64_t items = uem_cdiv(most_tiles(p.T, p.G, bm) * uem_cdiv(width, bn), 8) * 8;
    UEM_REQUIRE(items < ((int64_t)1 << 31), "%s: %lld tiles are more than a launch takes", what, (long long)items);
    if (bm == 256) go<T, FORM, 256, 256, 2, 4>(p, items, st);
    else if (bm == 128) go<T, FORM, 128, 128, 2, 2>(p, items, st);
    else go<T, FORM, 64, 128, 1, 4>(p, items, st);
    return uem_check_launch(what);
}

int check(const void* a, const void* b, const void* out, const void* offsets, int T, int G, int K, int N, int lda, int ldb, int flags, const char* what) {
    const int es = (flags & UEM_GROUPED_BF16) ? 2 : 4;
    UEM_REQUIRE(a && b && out && offsets, "%s: null pointer", what);
    UEM_REQUIRE(T > 0 && G > 0 && K > 0 && N > 0 && T < (1 << 30) && G < (1 << 16) && K <= (1 << 20) && N <= (1 << 20),
                "%s: rows < 2^30, groups < 65536, K and N <= 2^20 (got %d, %d, %d, %d)", what, T, G, K, N);
    UEM_REQUIRE((((uintptr_t)a | (uintptr_t)b) & 15) == 0 && (int64_t)lda * es % 16 == 0 && (int64_t)ldb * es % 16 == 0,
                "%s: operand rows must begin on 16-byte boundaries (uem_grouped_pad)", what);
    UEM_REQUIRE((int64_t)lda * es <= (1 << 23) && (int64_t)ldb * es <= (1 << 23), "%s: row strides of at most 8 MB", what);
    UEM_REQUIRE((flags & ~(UEM_GROUPED_BF16 | UEM_GROUPED_OUT_F32 | UEM_GROUPED_BIAS_BF16 | UEM_GROUPED_OFFSETS_64)) == 0, "%s: unknown flags %d", what, flags);
    return UEM_OK;
}
GgP params(const void* a, int lda, const void* b, int ldb, void* out, int ldo, const void* offsets, int T, int G, int K, int N, int flags) {
    GgP p{};
    const int es = (flags & UEM_GROUPED_BF16) ? 2 : 4;
    p.a = (const char*)a; p.b = (const char*)b; p.out = (char*)out; p.offsets = offsets;
    p.lda = (int64_t)lda * es; p.ldb = (int64_t)ldb * es; p.ldo = ldo; p.T = T; p.G = G; p.K = K; p.N = N;
    p.off64 = (flags & UEM_GROUPED_OFFSETS_64) != 0;
    p.bias16 = (flags & UEM_GROUPED_BIAS_BF16) != 0;
    p.out16 = (flags & UEM_GROUPED_BF16) && !(flags & UEM_GROUPED_OUT_F32);
    const int oes = p.out16 ? 2 : 4;
    p.vec = ((uintptr_t)out & 15) == 0 && (int64_t)ldo * oes % 16 == 0;
    return p;
}

}  // namespace

extern "C" int uem_grouped_pad(const void* src, int64_t src_ld, void* dst, int dst_ld, int cols, int64_t rows, int flags, void* stream) {
    UEM_REQUIRE(src && dst && rows > 0 && cols > 0 && dst_ld >= cols && src_ld >= cols, "grouped_pad: bad arguments");
    const int grid = uem_stream_grid(rows * dst_ld, 256);
    hipStream_t st = (hipStream_t)stream;
    if (flags & UEM_GROUPED_BF16) grouped_pad_kernel<bf16_t><<<grid, 256, 0, st>>>((const bf16_t*)src, src_ld, (bf16_t*)dst, dst_ld, cols, rows);
    else grouped_pad_kernel<float><<<grid, 256, 0, st>>>((const float*)src, src_ld, (float*)dst, dst_ld, cols, rows);
    return uem_check_launch("grouped_pad");
}
extern "C" int uem_grouped_fwd(const void* x, int x_ld, const void* w, int w_ld, const void* bias, void* y, const void* offsets, int T, int G, int K,
                               int N, int flags, void* stream) {
    const int rc = check(x, w, y, offsets, T, G, K, N, x_ld, w_ld, flags, "grouped_fwd");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(x_ld >= K && w_ld >= K, "grouped_fwd: row strides shorter than the rows");
    GgP p = params(x, x_ld, w, w_ld, y, N, offsets, T, G, K, N, flags);
    p.bias = bias;
    return (flags & UEM_GROUPED_BF16) ? launch_rows<bf16_t, FWD>(p, "grouped_fwd", (hipStream_t)stream)
                                      : launch_rows<float, FWD>(p, "grouped_fwd", (hipStream_t)stream);
}
extern "C" int uem_grouped_dgrad(const void* dy, int dy_ld, const void* w, int w_ld, void* dx, const void* offsets, int T, int G, int K, int N, int flags,
                                 void* stream) {
    const int rc = check(dy, w, dx, offsets, T, G, K, N, dy_ld, w_ld, flags, "grouped_dgrad");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(dy_ld >= N && w_ld >= K, "grouped_dgrad: row strides shorter than the rows");
    const GgP p = params(dy, dy_ld, w, w_ld, dx, K, offsets, T, G, K, N, flags);
    return (flags & UEM_GROUPED_BF16) ? launch_rows<bf16_t, DGRAD>(p, "grouped_dgrad", (hipStream_t)stream)
                                      : launch_rows<float, DGRAD>(p, "grouped_dgrad", (hipStream_t)stream);
}
extern "C" int64_t uem_grouped_wgrad_workspace_floats(int T, int G, int K, int N) {
    const int bm = wgrad_tile(G, N, K), chunk = wgrad_chunk(T, G, N, K, bm);
    // a group of m > 1 chunks has more than (m - 1) * chunk rows: at most 2 T / chunk slots in all
    const int64_t slots = T > chunk ? 2 * (int64_t)T / chunk : 0;
    const int64_t bias = ((int64_t)T / GG_BIAS_ROWS + G) * N;
    return (slots * (int64_t)N * K + 3) / 4 * 4 + bias;
}
extern "C" int uem_grouped_wgrad(const void* dy, int dy_ld, const void* x, int x_ld, void* dw, void* db, float* workspace, const void* offsets, int T,
                                 int G, int K, int N, int flags, void* stream) {
    const int rc = check(dy, x, dw ? dw : db, offsets, T, G, K, N, dy_ld, x_ld, flags, "grouped_wgrad");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(dy_ld >= N && x_ld >= K && workspace && ((uintptr_t)workspace & 15) == 0, "grouped_wgrad: bad row strides or workspace");
    hipStream_t st = (hipStream_t)stream;
    GgP p = params(dy, dy_ld, x, x_ld, dw, K, offsets, T, G, K, N, flags);
    const int bm = wgrad_tile(G, N, K);
    p.chunk = wgrad_chunk(T, G, N, K, bm);
    p.part = workspace;
    const int64_t slots = T > p.chunk ? 2 * (int64_t)T / p.chunk : 0;
    if (dw != nullptr) {
        const int64_t items = uem_cdiv((T / p.chunk + (int64_t)G) * uem_cdiv(N, bm) * uem_cdiv(K, bm), 8) * 8;
        UEM_REQUIRE(items < ((int64_t)1 << 31), "grouped_wgrad: %lld tiles are more than a launch takes", (long long)items);
        const bool h = (flags & UEM_GROUPED_BF16) != 0;
        if (bm == 256 && h) go<bf16_t, WGRAD, 256, 256, 2, 4>(p, items, st);
        else if (bm == 256) go<float, WGRAD, 256, 256, 2, 4>(p, items, st);
        else if (h) go<bf16_t, WGRAD, 128, 128, 2, 2>(p, items, st);
        else go<float, WGRAD, 128, 128, 2, 2>(p, items, st);
        if (slots > 0) {
            int64_t nb = uem_cdiv((int64_t)N * K, 256 * 4);
            grouped_join_kernel<<<dim3((unsigned)(nb < 1024 ? nb : 1024), (unsigned)G), 256, 0, st>>>(p);
        }
    }
    if (db != nullptr) {
        p.out = (char*)db;
        p.out16 = (flags & UEM_GROUPED_BIAS_BF16) != 0;
        p.part = workspace + (slots * (int64_t)N * K + 3) / 4 * 4;
        const int64_t items = (T / GG_BIAS_ROWS + (int64_t)G) * uem_cdiv(N, 64);
        if (flags & UEM_GROUPED_BF16) grouped_colsum_kernel<bf16_t><<<(unsigned)items, 256, 0, st>>>(p);
        else grouped_colsum_kernel<float><<<(unsigned)items, 256, 0, st>>>(p);
        grouped_colsum_join_kernel<<<dim3((unsigned)uem_cdiv(N, 256), (unsigned)G), 256, 0, st>>>(p);
    }
    return uem_check_launch("grouped_wgrad");
}
