// Products of feature rows with the weight of the group each row belongs to, the rows sorted by group and the groups' sizes known on the
// device only (offsets[g] .. offsets[g + 1] are the rows of group g):
//   forward          y[r]  = W_g x[r] + b_g         x [T][K], W [G][N][K], y [T][N]
//   data gradient    dx[r] = W_g^T dy[r]
//   weight gradient  dW_g  = sum over the group's rows of dy[r] x[r]^T,   db_g = sum of dy[r]
// Rows in front of offsets[0] and behind offsets[G] belong to no group: their y and dx are zeros and they enter no gradient.
//
// Matrix-bound (2 T K N flops each) once a group has some hundred rows, bound by reading W below.  One kernel serves the three: an
// operand tile travels global -> LDS by 16-byte LDS-DMA, 64 bytes of the reduction index per tile row a stage, five stages;
// where the reduction index is the SLOW one in memory (W in the data gradient, both operands of the weight gradient) the image is kept as
// it sits in memory and read transposed: bf16 by ds_read_b64_tr_b16, fp32 by consecutive ds_read_b32.  Both kinds are XOR-swizzled in
// 16-byte chunks on the source address so that a read covers all banks.  Buffer descriptors that end with the group's last row (and
// offsets beyond them for columns past the end) supply the zeros of every ragged edge: no row of another group is ever read.
// Products are exact in the fp32 accumulators (bf16) or fp32 MFMA (fp32); bf16 results are rounded once.
// Measured, bf16, 65536 x 2048 -> 2048 in 32 ragged groups, us: forward 485 - 520, data gradient 480 - 515, weight gradient with db 485 - 510
// (550 GFLOP each: 1.06 - 1.15 PFLOP/s; in groups of 2048 rows 470 = 1.17, a dense library product of the size 467): the clock falls to 1.7 GHz under the products, what
// is left is a tile's start and end.  fp32, 65536 x 2048 -> 2048 in 8 groups: 3.9 ms = 142 TFLOP/s of the 151 a dense product reaches.
//
// Nothing is read on the host: a block finds its tiles by prefix sums over the offsets, 64 groups to a wave, kept in registers.  Offsets are clamped to [0, T] and to the largest one in front of them, so that any
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
    void* db;                                     // WGRAD: column sums of dy, may be null
    float* part; float* part_db;                  // WGRAD: partial sums of groups of several row chunks
    const void* offsets;
    int64_t lda, ldb;                             // bytes of a row of a / of b
    int T, G, K, N, chunk;                        // K: columns of x (out of W's rows), N: columns of y;  chunk: rows of a WGRAD item
    int64_t ldo;                                  // elements of an output row
    bool off64, bias16, out16, vec;               // 64-bit offsets; bias or db / output in bf16; output rows take 16-byte stores
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
__device__ __forceinline__ int gg_offset(const GgP& p, int i) {
    int64_t o = p.off64 ? ((const int64_t*)p.offsets)[i] : (int64_t)((const int*)p.offsets)[i];
    o = o < 0 ? 0 : o;
    return (int)(o > p.T ? p.T : o);
}
// inclusive scans over a wave by DPP: inside the rows of 16 lanes, then the rows' totals carried on (a dozen cycles a step; by LDS exchange
// the two or three scans in front of a tile took 1 us)
template <int CTRL, int ROWS> __device__ __forceinline__ int lane_take(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ int scan_add(int v) {
    v += lane_take<0x111, 0xF>(0, v);              // row_shr 1, 2, 4, 8; lanes without a source take 0
    v += lane_take<0x112, 0xF>(0, v);
    v += lane_take<0x114, 0xF>(0, v);
    v += lane_take<0x118, 0xF>(0, v);
    v += lane_take<0x142, 0xA>(0, v);              // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v += lane_take<0x143, 0xC>(0, v);
    return v;
}
__device__ __forceinline__ int scan_max(int v) {   // v >= 0
    v = max(v, lane_take<0x111, 0xF>(0, v));
    v = max(v, lane_take<0x112, 0xF>(0, v));
    v = max(v, lane_take<0x114, 0xF>(0, v));
    v = max(v, lane_take<0x118, 0xF>(0, v));
    v = max(v, lane_take<0x142, 0xA>(0, v));
    v = max(v, lane_take<0x143, 0xC>(0, v));
    return v;
}
__device__ __forceinline__ int lane_value(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// The groups cut into tiles of `bm` rows, 64 groups at a time, one a lane, numbered in row order.
// LPT (the weight gradient's chunks): an empty group has a tile too (which writes its zeros), and the tiles are numbered whole ones first,
// then the groups' rests, the longest first: what comes last on the chip is short, however the rows fall to the groups.
struct Tile { int group, row0, rows, tile, tiles, slot; };        // rows, tiles: of the whole group
template <bool LPT>
struct Groups {
    int begin, len, nt, count, slots;             // of the lane's group; count, slots: tiles (LPT: whole ones) and slots up to and with it.
    bool rest;                                    // LPT: it has a tile that is not whole.  Groups of several tiles take as many slots
    int loaded;                                   // which 64 groups the lanes hold
    int first, last, total, rests;                // rows of all groups: [first, last); tiles (whole ones, rests) in all
    __device__ __forceinline__ void load(const GgP& p, int bm, int chunk, int lane, int& edge, int& before, int& nslot) {
        const int v = chunk * 64 + lane;
        int end = v < p.G ? gg_offset(p, v + 1) : 0;
        end = scan_max(end > edge ? end : edge);
        const int up = __shfl_up(end, 1, 64);
        begin = lane == 0 ? edge : up;
        len = end - begin;
        const int whole = v < p.G ? len / bm : 0;
        rest = v < p.G && (len > whole * bm || (LPT && len == 0));
        nt = whole + (rest ? 1 : 0);
        count = scan_add(LPT ? whole : nt) + before;
        slots = LPT ? scan_add(nt > 1 ? nt : 0) + nslot : 0;
        loaded = chunk;
        edge = lane_value(end, 63);
        before = lane_value(count, 63);
        nslot = LPT ? lane_value(slots, 63) : 0;
    }
    __device__ __forceinline__ void init(const GgP& p, int bm, int lane) {
        first = __builtin_amdgcn_readfirstlane(gg_offset(p, 0));
        last = first;
        total = rests = 0;
        int nslot = 0;
        for (int c = 0; c * 64 < p.G; ++c) {
            load(p, bm, c, lane, last, total, nslot);
            if (LPT) rests += __popcll(__ballot(rest));
        }
    }
    __device__ __forceinline__ Tile pick(int l) const {
        Tile t;
        t.group = loaded * 64 + l;
        t.row0 = lane_value(begin, l);
        t.rows = lane_value(len, l);
        t.tiles = lane_value(nt, l);
        t.slot = LPT ? lane_value(slots, l) - (t.tiles > 1 ? t.tiles : 0) : 0;
        t.tile = 0;
        return t;
    }
    // tile number `target` < total + rests
    __device__ __forceinline__ Tile find(const GgP& p, int bm, int lane, int target) {
        const bool is_rest = LPT && target >= total;
        if (is_rest) target -= total;
        if (p.G > 64) {                                                        // walk the groups 64 at a time again
            int edge = first, before = 0, nslot = 0;
            for (int c = 0; c * 64 < p.G; ++c) {
                load(p, bm, c, lane, edge, before, nslot);
                if (!is_rest && before > target) break;
                const int here = is_rest ? __popcll(__ballot(rest)) : 0;
                if (is_rest && here > target) break;
                target -= here;
            }
        }
        if (is_rest) {                                                         // the rest with `target` longer ones among the lanes'
            const int left = len - (nt - 1) * bm, key = rest ? (left < (1 << 25) ? left : (1 << 25) - 1) * 64 + 63 - lane : -1;
            const int n = p.G - loaded * 64 < 64 ? p.G - loaded * 64 : 64;
            int longer = 0;
            for (int i = 0; i < n; ++i) longer += lane_value(key, i) > key ? 1 : 0;
            Tile t = pick(__builtin_ctzll(__ballot(rest && longer == target)));
            t.tile = t.tiles - 1;
            return t;
        }
        const int l = __builtin_ctzll(__ballot(count > target));
        Tile t = pick(l);
        t.tile = target - (lane_value(count, l) - (LPT ? t.rows / bm : t.tiles));
        return t;
    }
    // the k-th of the groups of several tiles; false if there are not so many
    __device__ __forceinline__ bool several(const GgP& p, int bm, int lane, int k, Tile& t) {
        int edge = __builtin_amdgcn_readfirstlane(gg_offset(p, 0)), before = 0, nslot = 0;
        for (int c = 0; c * 64 < p.G; ++c) {
            load(p, bm, c, lane, edge, before, nslot);
            unsigned long long m = __ballot(nt > 1);
            const int here = __popcll(m);
            if (k >= here) { k -= here; continue; }
            for (; k > 0; --k) m &= m - 1;
            t = pick(__builtin_ctzll(m));
            return true;
        }
        return false;
    }
};
// Blocks go to the eight XCDs in turn: each XCD gets one contiguous run of the n items, neighbours share operand tiles in its L2.
__device__ __forceinline__ int xcd_item(int n) {
    const int x = blockIdx.x & 7, i = blockIdx.x >> 3, per = n >> 3, rem = n & 7;
    return i < per + (x < rem ? 1 : 0) ? x * per + (x < rem ? x : rem) + i : -1;
}

// Weight gradient: the tiles of a chunk cost what the chunk has rows, so each is spread over all eight XCDs (contiguous runs of the items, one an
// XCD, left the XCD with the longest groups behind: 65536 x 2048 x 2048 in 32 ragged groups 636 us, 555 spread; 7 classes 102 and 78): tile p of
// rt x ct goes to XCD p & 7, a rectangle of neighbours each where the sizes allow it, for what they share in its L2.
__device__ __forceinline__ int spread_tiles(int p, int rt, int ct) {
    const int x = p & 7, l = p >> 3;
    if ((rt & 3) == 0 && (ct & 1) == 0) return ((x >> 1) * (rt >> 2) + l / (ct >> 1)) * ct + (x & 1) * (ct >> 1) + l % (ct >> 1);
    if ((rt & 1) == 0 && (ct & 3) == 0) return ((x >> 2) * (rt >> 1) + l / (ct >> 2)) * ct + (x & 3) * (ct >> 2) + l % (ct >> 2);
    return p;
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
    // piece j of stage `q`, all of whose reduction indices exist (a KC row past the operand's end lies past the descriptor's)
    __device__ __forceinline__ void issue_whole(int j, const i32x4 rs, char* img, int wave, int q) const {
        uem_raw_buffer_load_lds(rs, (lds_u32p)(img + (j * NW + wave) * 1024), 16, (int)off[j], KS ? 0 : q * 64, 0, 0);
    }
    // piece j of stage `q` of a reduction of `red`
    __device__ __forceinline__ void issue(int j, const i32x4 rs, char* img, int wave, int q, int red) const {
        const unsigned o = KS ? off[j] : (q * (64 / ES) + kc[j] < red ? off[j] + (unsigned)q * 64u : GG_OOB);
        uem_raw_buffer_load_lds(rs, (lds_u32p)(img + (j * NW + wave) * 1024), 16, (int)o, 0, 0, 0);
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
// a lane's elements of a fragment added to s, on the vector units (bf16 two at a time, as products with ones: 517 us where eight unpacked
// additions took 544, 65536 x 2048 x 2048 with db in 32 groups; without db 494)
template <typename FA> __device__ __forceinline__ float add_of(const FA& a, float s, bf16_t) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a.v[2 * i], a.v[2 * i + 1]}, ones, s, false);
    return s;
}
template <typename FA> __device__ __forceinline__ float add_of(const FA& a, float s, float) { return s + ((a.v[0] + a.v[1]) + (a.v[2] + a.v[3])); }
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

// Rows of no group: zeros.  Shared out over the blocks without one of the n items (there are as a rule as many as such rows make tiles; they come
// last, when CUs run out of items: 32768 rows x 512, half of them of no group, 21.5 -> 19.4 us; a fifth, x 512 of 2048, 70.5 -> 68.5; at worst
// 65536 x 1024, half of them, 80.3 -> 82.5), or over all if there is none.
template <int NTH>
__device__ __forceinline__ void zero_rows(const GgP& p, const Groups<false>& groups, int width, int n) {
    const int head = groups.first, zeros = head + p.T - groups.last, free = (int)gridDim.x - n;
    int z = blockIdx.x, step = gridDim.x;
    if (free > 0) {
        const int x = blockIdx.x & 7, i = blockIdx.x >> 3, per = n >> 3, rem = n & 7;
        const int late = i - per - (x < rem ? 1 : 0);                          // its place among its XCD's blocks without an item
        if (late < 0) return;
        z = x * ((int)(gridDim.x >> 3) - per) - (x < rem ? x : rem) + late;
        step = free;
    }
    for (; z < zeros; z += step) {
        const int64_t at = (int64_t)(z < head ? z : groups.last + z - head) * p.ldo;
        if (p.vec) {
            const int n = p.out16 ? 8 : 4;
            for (int c = threadIdx.x * n; c < width; c += NTH * n) *reinterpret_cast<uint4*>(p.out + (at + c) * (p.out16 ? 2 : 4)) = make_uint4(0, 0, 0, 0);
        } else {
            for (int c = threadIdx.x; c < width; c += NTH)
                if (p.out16) reinterpret_cast<bf16_t*>(p.out)[at + c] = 0;
                else reinterpret_cast<float*>(p.out)[at + c] = 0.f;
        }
    }
}
template <int NTH> __device__ __forceinline__ void zero_rows(const GgP&, const Groups<true>&, int, int) {}

// One tile a block.  Five stages: while stage t is computed on, a KS operand's pieces of stage t + 4 leave, a KC operand's of stages t + 3 and
// t + 4 together if t is odd -- the two halves of every 128-byte line one after the other, or the line travels from L2 twice (65536 x 2048 ->
// 2048 in 32 groups, forward: 545 us stage by stage, 515 in pairs; KS operands in pairs lose: weight gradient 488 against 529).
// PP (eight waves, one block a CU): the two waves of a SIMD take turns -- while one feeds the matrix cores from registers, the other reads
// its next fragments and sends pieces off, a barrier between the turns.  With the waves in step both wait for LDS at the same time.
// The MFMA's rows are the output's COLUMNS (its A operand is tile b): a lane ends up with four neighbouring columns of one row.
template <typename T, int FORM, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void grouped_kernel(const GgP p) {
    constexpr int ES = sizeof(T), NW = WGM * WGN, MT = BM / WGM / 32, NT = BN / WGN / 32, BK = 64 / ES, SB = (BM + BN) * 64, NST = 5;
    constexpr bool PP = NW == 8, AKS = FORM == WGRAD, BKS = FORM != FWD;
    using LA = Loader<T, AKS, BM, NW>;
    using LB = Loader<T, BKS, BN, NW>;
    constexpr bool SPLIT = PP && !AKS && !BKS && LB::IPW % 2 == 0;       // both operands KC: b's pairs leave in halves
    constexpr int FLIGHT_EVEN = 2 * LA::IPW + LB::IPW;                         // SPLIT, in front of an even stage
    constexpr int FLIGHT = LA::IPW * (AKS ? 3 : 2) + LB::IPW * (BKS ? 3 : 2);
    constexpr int ROWB = NT * 64, CPR = ROWB / 16;                             // bf16 results: bytes and 16-byte chunks of a wave's row
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bm = FORM == WGRAD ? p.chunk : BM;                               // feature rows of a tile / of a chunk
    const int width = FORM == FWD ? p.N : p.K;                                 // output columns
    const int ct = (width + BN - 1) / BN, rt = FORM == WGRAD ? (p.N + BM - 1) / BM : 1;
    Groups<FORM == WGRAD> groups;
    groups.init(p, bm, lane);

    if (FORM != WGRAD) zero_rows<64 * NW>(p, groups, width, groups.total * ct);
    const int item = FORM == WGRAD ? ((int)blockIdx.x < (groups.total + groups.rests) * ct * rt ? (int)blockIdx.x : -1) : xcd_item(groups.total * ct * rt);
    if (item < 0) return;

    // ---- the tile
    const Tile tl = groups.find(p, bm, lane, item / (ct * rt));
    int within = item % (ct * rt);
    if (FORM == WGRAD) within = spread_tiles(within, rt, ct);
    const int c0 = (within % ct) * BN, n0 = (within / ct) * BM;                // n0: first row of W (WGRAD)
    const int r0 = tl.row0 + tl.tile * bm;
    int rows = tl.rows - tl.tile * bm;                                         // feature rows of the tile
    rows = rows < 0 ? 0 : rows < bm ? rows : bm;
    const int red = FORM == FWD ? p.K : FORM == DGRAD ? p.N : rows;            // reduction length
    const int steps = (red + BK - 1) / BK;
    LA la;
    LB lb;
    la.init(wave, lane, p.lda, n0, p.N);
    lb.init(wave, lane, p.ldb, c0, p.K);
    const char* pa = p.a + (int64_t)r0 * p.lda;
    const char* pb = FORM == FWD ? p.b + ((int64_t)tl.group * p.N + c0) * p.ldb : FORM == DGRAD ? p.b + (int64_t)tl.group * p.N * p.ldb : p.b + (int64_t)r0 * p.ldb;
    // bytes of a row, up to the 16-byte boundary behind its last element (zeros there)
    const unsigned acols = (unsigned)((FORM == FWD ? p.K : p.N) * ES + 15) & ~15u, bcols = (unsigned)(p.K * ES + 15) & ~15u;
    int arem = rows, brem = FORM == FWD ? (p.N - c0 < BN ? p.N - c0 : BN) : FORM == DGRAD ? p.N : rows;       // rows left of a and b
    const int wm = (wave / WGN) * (MT * 32), wn = (wave % WGN) * (NT * 32);
    float bias = 0.f;                                                          // of column wn + lane
    if (FORM == FWD && p.bias != nullptr) {
        const int c = c0 + wn + lane;
        const int64_t i = (int64_t)tl.group * p.N + c;
        if (lane < NT * 32 && c < p.N) bias = p.bias16 ? __uint_as_float((uint32_t)((const bf16_t*)p.bias)[i] << 16) : ((const float*)p.bias)[i];
    }

    // One operand's stage `q`, or stages `q` and `q` + 1; those past the end fetch zeros, so that the waits' counts hold.
    // Stages that lie wholly inside the reduction are sent without a check a lane, by the eight waves alone: 65536 x 2048 x 2048
    // in 32 groups gains 1 to 2 %, and the four waves' schedule, which has no phase of its own for it, loses 5 to 8 %.
    auto desc = [](const char* b, int rem, int64_t ld, unsigned bytes, bool ks) {
        const int n = ks && rem > BK ? BK : rem;
        return rsrc(b, n > 0 ? (unsigned)((n - 1) * ld) + bytes : 0u);
    };
    int qa = 0, qb = 0;                                                        // next stages to send off
    auto issue_a = [&](char* __restrict__ fill0, char* __restrict__ fill1, const bool two) {
        const i32x4 r0_ = desc(pa, arem, p.lda, acols, AKS);
        if (AKS || (PP && (qa + (two ? 2 : 1)) * BK <= red)) {
#pragma unroll
            for (int j = 0; j < LA::IPW; ++j) {
                la.issue_whole(j, r0_, fill0, wave, qa);
                if (two) la.issue_whole(j, r0_, fill1, wave, qa + 1);
            }
        } else {
#pragma unroll
            for (int j = 0; j < LA::IPW; ++j) {
                la.issue(j, r0_, fill0, wave, qa, red);
                if (two) la.issue(j, r0_, fill1, wave, qa + 1, red);
            }
        }
        if (AKS) { pa += BK * p.lda; arem -= BK; }
        qa += two ? 2 : 1;
    };
    auto issue_b = [&](char* __restrict__ fill0, char* __restrict__ fill1, const bool two, const int first, const int end) {
        const i32x4 r0_ = desc(pb, brem, p.ldb, bcols, BKS);
        if (BKS || (PP && (qb + (two ? 2 : 1)) * BK <= red)) {
#pragma unroll
            for (int j = first; j < end; ++j) {
                lb.issue_whole(j, r0_, fill0 + BM * 64, wave, qb);
                if (two) lb.issue_whole(j, r0_, fill1 + BM * 64, wave, qb + 1);
            }
        } else {
#pragma unroll
            for (int j = first; j < end; ++j) {
                lb.issue(j, r0_, fill0 + BM * 64, wave, qb, red);
                if (two) lb.issue(j, r0_, fill1 + BM * 64, wave, qb + 1, red);
            }
        }
        if (end < LB::IPW) return;
        if (BKS) { pb += BK * p.ldb; brem -= BK; }
        qb += two ? 2 : 1;
    };
    // in stage t: a KC operand's stages t + 3 and t + 4 if t is odd (SPLIT: of b half their pieces, the other half in the stage behind; with all of
    // both operands in the odd stages 65536 x 2048 -> 2048 in 32 groups took 500 us, so 470), a KS operand's stage t + 4
    auto issue = [&](char* __restrict__ fill2, char* __restrict__ fill3, char* __restrict__ fill4, const bool odd) {
        if (AKS) issue_a(fill4, fill4, false);
        else if (odd) issue_a(fill3, fill4, true);
        if (BKS) issue_b(fill4, fill4, false, 0, LB::IPW);
        else if (!SPLIT) { if (odd) issue_b(fill3, fill4, true, 0, LB::IPW); }
        else if (odd) issue_b(fill3, fill4, true, 0, LB::IPW / 2);
        else issue_b(fill2, fill3, true, LB::IPW / 2, LB::IPW);
    };
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    // db: the blocks of W's first columns also add up dy's columns, one fragment of them a wave
    const bool sums = FORM == WGRAD && p.db != nullptr && c0 == 0;
    static_assert(FORM != WGRAD || MT == WGN, "a wave for each fragment of dy's columns");
    float colsum = 0.f;
    Frag<T, AKS, BM> fa[2][MT];
    Frag<T, BKS, BN> fb[2][NT];
    // one function with the stages being refilled and the stage being read as __restrict__ pointers: that is what tells the compiler that
    // the reads do not depend on the LDS-DMA in flight (it would wait for all of it in front of the first read)
    auto stage = [&](char* __restrict__ fill2, char* __restrict__ fill3, char* __restrict__ fill4, const char* __restrict__ use, const bool odd) {
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
                for (int j = 0; j < NT; ++j) mma(fb[ks][j], fa[ks][i], acc[i][j], T{});
        };
        auto add_up = [&]() {                                                  // away from the MFMAs: a branch among them costs 15 % of all blocks' time
            if (!sums) return;
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (i == wave % WGN) colsum = add_of(fa[1][i], add_of(fa[0][i], colsum, T{}), T{});
        };
        // In front of stage t (PP: in stage t - 1, behind its sends) the pieces of stage t have to have landed.  Newer than the last of them
        // are, of a KS operand, three stages' pieces and, of a KC operand, those of the pair behind its own (and, t even, its partner's last;
        // SPLIT, t even: what one odd stage sends; t odd: that and the halves of the even stage behind it).
        if (PP) {
            fetch(0);
            fetch(1);
            __builtin_amdgcn_sched_barrier(0);                                 // the reads first: the sends' addresses are made in their shadow
            issue(fill2, fill3, fill4, odd);
            if (SPLIT && odd) gg_wait<FLIGHT_EVEN>();
            else gg_wait<FLIGHT>();
            if (FORM == WGRAD) add_up();
            gg_barrier();
            __builtin_amdgcn_s_setprio(1);
            multiply(0);
            multiply(1);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            gg_barrier();
        } else {
            gg_wait<FLIGHT>();
            gg_barrier();
            issue(fill2, fill3, fill4, odd);
            fetch(0);
            fetch(1);
            multiply(0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(1);
            if (FORM == WGRAD) add_up();
        }
    };
    if (steps > 0) {
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
            char* const f0 = smem + t * SB;
            char* const f1 = f0 + SB;
            if (!AKS) issue_a(f0, f1, true);
            if (!BKS) issue_b(f0, f1, true, 0, SPLIT && t == 2 ? LB::IPW / 2 : LB::IPW);
            if (AKS) issue_a(f0, f0, false);
            if (BKS) issue_b(f0, f0, false, 0, LB::IPW);
            if (AKS) issue_a(f1, f1, false);
            if (BKS) issue_b(f1, f1, false, 0, LB::IPW);
        }
        if (PP) {
            if (SPLIT) gg_wait<FLIGHT_EVEN>();
            else gg_wait<FLIGHT>();
            gg_barrier();
            if (wave >= NW / 2) gg_barrier();
        }
        int u = 0;                                                             // stage t's place in the ring
        auto place = [](int k) { return (k >= NST ? k - NST : k) * SB; };
        for (int t = 0; t < steps; t += 2) {                                   // an odd number of stages: the last one multiplies zeros
            stage(smem + place(u + 2), smem + place(u + 3), smem + place(u + 4), smem + u * SB, false);
            stage(smem + place(u + 3), smem + place(u + 4), smem + u * SB, smem + place(u + 1), true);
            u = u + 2 >= NST ? u + 2 - NST : u + 2;
        }
        if (PP && wave < NW / 2) gg_barrier();
    }
    gg_wait<0>();                                                              // everybody has read the last stage and nothing is on its way:
    gg_barrier();                                                              // the stages' memory takes the results

    // ---- results
    const bool partial = FORM == WGRAD && tl.tiles > 1;                   // a chunk of a group with several: to its slot, in fp32
    const int64_t ldo = FORM == WGRAD ? p.K : p.ldo;
    const int64_t first = (FORM == WGRAD ? (int64_t)(partial ? tl.slot + tl.tile : tl.group) * p.N * p.K + (int64_t)n0 * ldo : (int64_t)r0 * ldo) + wm * ldo + c0 + wn;
    const int left = (FORM == WGRAD ? p.N - n0 : rows) - wm, cols = width - c0 - wn;            // output rows and columns from the wave's first on
    char* const out = partial ? (char*)p.part : p.out;
    const int fr = lane & 31, fh = lane >> 5;
    if (FORM == WGRAD) colsum += __shfl_xor(colsum, 32, 64);                    // the two halves of the wave hold other rows
    if (sums && fh == 0) {
        const int n = n0 + wm + (wave % WGN) * 32 + fr;
        if (n < p.N) {
            if (partial) p.part_db[(int64_t)(tl.slot + tl.tile) * p.N + n] = colsum;
            else if (p.bias16) ((bf16_t*)p.db)[(int64_t)tl.group * p.N + n] = (bf16_t)bf_bits(colsum);
            else ((float*)p.db)[(int64_t)tl.group * p.N + n] = colsum;
        }
    }
    // a lane's accumulators 4 h .. 4 h + 3 of fragment (i, j): columns j * 32 + 8 h + 4 fh + 0 .. 3 of row i * 32 + fr
    if (FORM == FWD && p.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float b = __shfl(bias, j * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh, 64);
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i][j][r] += b;
            }
    }
    if (!partial && p.out16) {
        char* const mine = smem + wave * MT * 32 * ROWB;                       // the wave's result rows, to leave as whole 16-byte chunks
        static_assert(NW * MT * 32 * ROWB <= NST * SB, "the results in the stages' memory");
        auto slot = [&](int row, int chunk) { return mine + row * ROWB + ((chunk ^ (CPR == 8 ? (row >> 1) & 7 : (row >> 2) & 3)) << 4); };
        bf16_t* const dst = reinterpret_cast<bf16_t*>(out) + first;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const f32x16& a = acc[i][j];
                    *reinterpret_cast<uint2*>(slot(i * 32 + fr, j * 4 + h) + fh * 8) = make_uint2(bf_bits(a[4 * h]) | (bf_bits(a[4 * h + 1]) << 16),
                                                                                                 bf_bits(a[4 * h + 2]) | (bf_bits(a[4 * h + 3]) << 16));
                }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                     // the wave's own rows, written by all its lanes
        if (p.vec) {                                                           // streamed: nothing of this launch reads them (12 % of short reductions' time)
#pragma unroll
            for (int t = 0; t < MT * 32; t += 64 / CPR) {
                const int row = t + lane / CPR, ch = lane % CPR;
                if (row < left && ch * 8 < cols)
                    __builtin_nontemporal_store(*reinterpret_cast<const f32x4*>(slot(row, ch)), reinterpret_cast<f32x4*>(dst + row * ldo + ch * 8));
            }
        } else {
            for (int t = lane; t < MT * 32 * NT * 32; t += 64) {
                const int row = t / (NT * 32), c = t % (NT * 32);
                if (row < left && c < cols) dst[row * ldo + c] = *reinterpret_cast<const bf16_t*>(slot(row, c >> 3) + (c & 7) * 2);
            }
        }
    } else {
        float* const dst = reinterpret_cast<float*>(out) + first;
        const bool vec = partial ? (p.K & 3) == 0 : p.vec;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const f32x16& a = acc[i][j];
                    const int c = j * 32 + 8 * h + 4 * fh;
                    if (i * 32 + fr >= left) continue;
                    float* const d = dst + (i * 32 + fr) * ldo + c;
                    if (vec) {
                        if (c < cols) *reinterpret_cast<f32x4*>(d) = f32x4{a[4 * h], a[4 * h + 1], a[4 * h + 2], a[4 * h + 3]};
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < cols) d[e] = a[4 * h + e];
                    }
                }
    }
}

// The forward and the data gradient of a few rows: the weights' bytes are all there is, and the latency of reaching them.  A tile is 32 rows x
// 32 columns, its reduction shared out over sixteen waves that load their fragments straight into registers -- at 2048 channels a wave has all
// of its 8 KB of W on the way at once -- and are joined through LDS in wave order.  The data gradient's fragments of W are gathered element by
// element, neighbouring lanes from neighbouring addresses.  Rows may begin on any element: a copy of W to padded rows would cost its bytes twice
// over (one row, 27 groups, 1358 -> 1414 bf16, a training step 147 us, so 85).  Nine rows in six groups, 2048 -> 512: 13.5 -> 7.2 us.
template <typename T, int FORM>
__global__ __launch_bounds__(1024) void grouped_few_kernel(const GgP p) {
    constexpr int ES = sizeof(T), PER = 16 / ES, NW = 16, LD = 36, DEEP = FORM == FWD ? 8 : 4;        // LD: floats of a staged row, off the bank period
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    struct __attribute__((packed, aligned(ES))) Chunk { unsigned w[4]; };                             // 16 bytes of a row, on any element boundary
    auto chunk = [](const char* q) {
        const Chunk c = *reinterpret_cast<const Chunk*>(q);
        return u32x4{c.w[0], c.w[1], c.w[2], c.w[3]};
    };
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* const red = reinterpret_cast<float*>(smem);
    const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int width = FORM == FWD ? p.N : p.K, length = FORM == FWD ? p.K : p.N;
    Groups<false> groups;
    groups.init(p, 32, lane);
    const int ct = (width + 31) / 32, item = xcd_item(groups.total * ct);
    zero_rows<1024>(p, groups, width, groups.total * ct);
    if (item < 0) return;
    const Tile tl = groups.find(p, 32, lane, item / ct);
    const int c0 = (item % ct) * 32, r0 = tl.row0 + tl.tile * 32, rows = min(32, tl.rows - tl.tile * 32);
    // lanes of rows and columns past the end read the last one again; their results are not stored
    const char* const px = p.a + (int64_t)(r0 + min(fr, rows - 1)) * p.lda;
    const int c = min(c0 + fr, width - 1);
    const char* const pw = FORM == FWD ? p.b + ((int64_t)tl.group * p.N + c) * p.ldb : p.b + (int64_t)tl.group * p.N * p.ldb + c * ES;
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    const int steps = (length + 2 * PER - 1) / (2 * PER);                      // a lane's 16 bytes are chunk 2 * step + fh
    for (int s0 = wave; s0 < steps; s0 += NW * DEEP) {
        Frag<T, false, 32> x[DEEP], w[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            // the last chunk that lies inside the row stands in for those past its end, without what the chunk in front of it holds already
            if (s0 + k * NW >= steps) continue;
            const int from = min((2 * (s0 + k * NW) + fh) * PER, length - PER);
            x[k].v = __builtin_bit_cast(decltype(x[k].v), chunk(px + from * ES));
            if (FORM == FWD) w[k].v = __builtin_bit_cast(decltype(w[k].v), chunk(pw + from * ES));
            else {
                struct { T e[PER]; } c;
#pragma unroll
                for (int e = 0; e < PER; ++e) c.e[e] = *reinterpret_cast<const T*>(pw + (int64_t)(from + e) * p.ldb);
                w[k].v = __builtin_bit_cast(decltype(w[k].v), c);
            }
        }
        __builtin_amdgcn_sched_barrier(0);                                     // all of them on their way before the first is waited for
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            if (s0 + k * NW != steps - 1) continue;                            // (uniform) the chunks of both halves exist, or neither
            const int at = (2 * (s0 + k * NW) + fh) * PER, skip = at - min(at, length - PER);
            u32x4 keep;
#pragma unroll
            for (int j = 0; j < 4; ++j) keep[j] = ES == 4 ? (j >= skip ? ~0u : 0u) : (2 * j >= skip ? 0xffffu : 0u) | (2 * j + 1 >= skip ? 0xffff0000u : 0u);
            x[k].v = __builtin_bit_cast(decltype(x[k].v), __builtin_bit_cast(u32x4, x[k].v) & keep);
            w[k].v = __builtin_bit_cast(decltype(w[k].v), __builtin_bit_cast(u32x4, w[k].v) & keep);
        }
#pragma unroll
        for (int k = 0; k < DEEP; ++k)
            if (s0 + k * NW < steps) mma(w[k], x[k], acc, T{});
    }
#pragma unroll
    for (int h = 0; h < 4; ++h)                                                // rows of the result: columns 8 h + 4 fh + 0 .. 3 of feature row fr
        *reinterpret_cast<f32x4*>(red + (wave * 32 + fr) * LD + 8 * h + 4 * fh) = f32x4{acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]};
    __syncthreads();
    const int m = threadIdx.x >> 5, n = threadIdx.x & 31;
    if (m >= rows || c0 + n >= width) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[(w * 32 + m) * LD + n];
    if (p.bias != nullptr) {
        const int64_t i = (int64_t)tl.group * p.N + c0 + n;
        v += p.bias16 ? __uint_as_float((uint32_t)((const bf16_t*)p.bias)[i] << 16) : ((const float*)p.bias)[i];
    }
    const int64_t at = (int64_t)(r0 + m) * p.ldo + c0 + n;
    if (p.out16) reinterpret_cast<bf16_t*>(p.out)[at] = (bf16_t)bf_bits(v);
    else reinterpret_cast<float*>(p.out)[at] = v;
}

// the sum of n values `step` apart, in their order, four of them on the way at a time
template <typename V> __device__ __forceinline__ V sum_in_order(const V* p, int64_t step, int n) {
    V v = *p;
    for (int c = 1; c < n; c += 4) {
        V u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = c + k < n ? p[(c + k) * step] : V{};
#pragma unroll
        for (int k = 0; k < 4; ++k) v += u[k];
    }
    return v;
}
// store(i, sum of src[i], src[i + step] ... n of them) for i < count, by the block `block` of `blocks`.  Many chunks are shared out over 4 or 16
// slices of the block, whose sums are added in order (65536 rows, 64 -> 32 in one group, 256 chunks: 40 us by one thread an
// element, 5 so)
template <typename V, typename S> __device__ __forceinline__ void join_sums(const V* src, int64_t count, int64_t step, int n, int block, int blocks, V* red, S store) {
    const int slices = n > 64 ? 16 : n > 16 ? 4 : 1, lanes = 256 / slices, l = threadIdx.x % lanes, sl = threadIdx.x / lanes;
    const int c0 = (int)((int64_t)n * sl / slices), c1 = (int)((int64_t)n * (sl + 1) / slices);
    for (int64_t base = (int64_t)block * lanes; base < count; base += (int64_t)blocks * lanes) {
        const int64_t i = base + l;
        V v{};
        if (i < count) v = sum_in_order(src + c0 * step + i, step, c1 - c0);
        if (slices > 1) {
            red[threadIdx.x] = v;
            __syncthreads();
            if (sl == 0)
                for (int k = 1; k < slices; ++k) v += red[k * lanes + l];
            __syncthreads();
        }
        if (sl == 0 && i < count) store(i, v);
    }
}
// dW and db of the groups of several chunks = their partial sums, added in a fixed order.  blockIdx.y: which of those groups; the last blockIdx.x: db
__global__ __launch_bounds__(256) void grouped_join_kernel(const GgP p) {
    __shared__ f32x4 red[256];
    Tile t{};
    Groups<true> groups;
    if (!groups.several(p, p.chunk, threadIdx.x & 63, blockIdx.y, t)) return;
    const int g = t.group, n = t.tiles, blocks = gridDim.x - 1;
    const int64_t size = (int64_t)p.N * p.K;
    const float* const part = p.part + t.slot * size;
    if ((int)blockIdx.x == blocks) {
        if (p.db == nullptr) return;
        join_sums(p.part_db + (int64_t)t.slot * p.N, p.N, p.N, n, 0, 1, reinterpret_cast<float*>(red), [&](int64_t c, float v) {
            if (p.bias16) ((bf16_t*)p.db)[(int64_t)g * p.N + c] = (bf16_t)bf_bits(v);
            else ((float*)p.db)[(int64_t)g * p.N + c] = v;
        });
    } else if (p.vec && (size & 3) == 0) {                                     // rows of whole 16-byte stores: so is the whole of dW_g
        join_sums(reinterpret_cast<const f32x4*>(part), size / 4, size / 4, n, blockIdx.x, blocks, red, [&](int64_t i, const f32x4 v) {
            if (p.out16) *reinterpret_cast<uint2*>(p.out + (g * size + 4 * i) * 2) = make_uint2(bf_bits(v[0]) | (bf_bits(v[1]) << 16), bf_bits(v[2]) | (bf_bits(v[3]) << 16));
            else *reinterpret_cast<f32x4*>(p.out + (g * size + 4 * i) * 4) = v;
        });
    } else {
        join_sums(part, size, size, n, blockIdx.x, blocks, reinterpret_cast<float*>(red), [&](int64_t i, float v) {
            if (p.out16) reinterpret_cast<bf16_t*>(p.out)[g * size + i] = (bf16_t)bf_bits(v);
            else reinterpret_cast<float*>(p.out)[g * size + i] = v;
        });
    }
}

// dst[r][0 .. 8 cpr) = src[r][0 .. cols), zeros behind: rows that begin on 16-byte boundaries (cpr chunks of 16 bytes each, one a thread)
template <typename T>
__global__ __launch_bounds__(256) void grouped_pad_kernel(const T* __restrict__ src, int64_t lds, T* __restrict__ dst, int cpr, int cols, int64_t chunks) {
    constexpr int PER = 16 / sizeof(T);
    struct __attribute__((aligned(16))) Chunk { T e[PER]; };
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t r = chunks < ((int64_t)1 << 31) ? (int64_t)((uint32_t)i / (uint32_t)cpr) : i / cpr;
        const int c = (int)(i - r * cpr) * PER;
        const T* const p = src + r * lds + c;
        Chunk v;
#pragma unroll
        for (int k = 0; k < PER; ++k) v.e[k] = c + k < cols ? p[k] : (T)0;
        reinterpret_cast<Chunk*>(dst)[i] = v;
    }
}

template <typename T, int FORM, int BM, int BN, int WGM, int WGN>
int go(const GgP& p, int64_t items, const char* what, hipStream_t st) {
    constexpr int LDS = 5 * (BM + BN) * 64, THREADS = 64 * WGM * WGN;
    const int64_t blocks = uem_cdiv(items, 8) * 8;
    UEM_REQUIRE(blocks * THREADS < ((int64_t)1 << 32), "%s: %lld tiles of %d threads are more than a launch holds (2^32 threads)", what, (long long)items, THREADS);
    auto k = grouped_kernel<T, FORM, BM, BN, WGM, WGN>;
    if (!uem_allow_lds((const void*)k, LDS)) return uem_check_launch(what);
    k<<<(unsigned)blocks, THREADS, LDS, st>>>(p);
    return uem_check_launch(what);
}

// Tile of the forward and the data gradient: the one whose slowest CU has the least to do.  The larger a tile the fewer operand bytes a
// flop; a smaller one wastes less of a short group and spreads further.  The factors are the rates measured with every CU at work, of the
// best tile's: bf16 65536 x 2048 -> 2048 in 32 groups 500 / 597 / 845 us; fp32 65536 x 1024 -> 2048 in 32 groups 2090 / 1997 / 2104 us, and
// at no size tried has the largest been the best in fp32 (26214 x 512 -> 512 in 7 groups 136 / 134 / 124): it is not built.
struct TileShape { int bm, bn; double rate16, rate32; };
constexpr TileShape TILES[3] = {{256, 256, 1.0, 0.0}, {128, 128, 0.8, 1.0}, {64, 128, 0.6, 0.97}};
int64_t likely_tiles(int T, int G, int bm) { return uem_cdiv(T, bm) + (G < T ? G : T) / 2; }      // half a tile of each group is empty
int pick_tile(int T, int G, int width, bool is16) {
    int best = -1;
    double least = 0;
    for (int i = is16 ? 0 : 1; i < 3; ++i) {
        const double n = (double)uem_cdiv(likely_tiles(T, G, TILES[i].bm) * uem_cdiv(width, TILES[i].bn), 256);
        const double cost = n * TILES[i].bm * TILES[i].bn / (is16 ? TILES[i].rate16 : TILES[i].rate32);
        if (best < 0 || cost < least) { best = i; least = cost; }
    }
    return best;
}
// Tiles of the weight gradient.  fp32: 128 x 128, two of them a CU (its products are slow enough that the larger tile's fewer operand bytes
// gain nothing and its rounding up of N, K and the blocks' number costs up to half: 40000 x (640 -> 768) in 13 groups 682 / 340 us).
// bf16: 256 x 256 where each of the 256 CUs has the products of 1536 rows of such a tile to do: 65536 x 2048 x 2048 in 32 groups 504 us / 618 with
// 128 x 128, 60000 x (640 -> 768) in 5 97 / 142 (2109 rows a CU); 20000 x 1024 x 1024 in 24 76 / 60 (1250), 9000 x (2048 -> 1024) in 12 65 / 52 (1125).
int wgrad_tile(int T, int N, int K, bool is16) { return is16 && (int64_t)T * uem_cdiv(N, 256) * uem_cdiv(K, 256) >= 1536 * 256 && N > 128 && K > 128 ? 256 : 128; }
// Rows of a weight-gradient item: what one of the 256 blocks at work (two of them a CU with 128 x 128 tiles) has to do in all, so that a group with
// most of the rows spreads over the chip; each slot of partial sums costs N * K * 8 bytes of traffic.  With 256 x 256 tiles a block too many is a
// round too many: each group's rest counts as half an item, in as many rounds as leave room for the others.  32768 x (2048 -> 512) in 7 groups
// 101 -> 91 us, 60000 x (640 -> 768) in 5 108 -> 97; with 128 x 128 tiles it loses as often as it gains.
int wgrad_chunk(int T, int G, int N, int K, int bm) {
    const double per = (bm == 256 ? 256. : 512.) / (double)(uem_cdiv(N, bm) * uem_cdiv(K, bm));        // items of a tile in a round
    double n = per;
    if (bm == 256) {
        const double rests = 0.5 * (G < T ? G : T);
        n = ceil(rests / per + 0.5) * per - rests;
    }
    const int64_t c = (int64_t)ceil(T / n);
    return (int)(uem_cdiv(c < 256 ? 256 : c < T ? c : T, 64) * 64);
}
int64_t wgrad_slots(int T, int chunk) { return T > chunk ? 2 * (int64_t)T / chunk : 0; }      // m > 1 chunks are of more than (m - 1) * chunk rows

// 32 x 32 tiles of sixteen waves: while they are few -- the larger tiles would leave most CUs idle, each block walking the whole reduction -- and
// rows are long enough to share out.  Measured, us, the larger tiles / these, with these tiles' number in brackets:
//   bf16 forward 2048 -> 512 14.8 / 7.4 (64), 14.8 / 10.2 (176), 15.0 / 18.6 (400); 1024 -> 1024 9.0 / 7.7 (384); 512 -> 512 6.1 / 5.1 (176);
//     64 -> 1024 3.8 / 5.6 (160).  Data gradient, reduction 2048 14.6 / 7.8 (48), 15.0 / 16.8 (408); 1024 9.2 / 6.7 (192); 512 6.4 / 4.9 (80),
//     6.9 / 8.3 (256); 256 5.4 / 7.6 (160).
//   fp32 forward 2048 -> 512 72 / 25 (176), 74 / 66 (800), 76 / 126 (1552); 1024 -> 1024 38 / 14 (384), 40 / 35 (832); 512 -> 512 22 / 17 (400),
//     22 / 27 (800); 256 -> 2048 11.5 / 7.2 (64), 11.6 / 13.0 (320); 64 -> 1024 5.2 / 8.5 (160).  Data gradient alike: 2048 72 / 21 (208), 1024 38 / 11 (54).
bool few_rows(int64_t tiles, int length, bool is16, bool dgrad) {
    if (is16) return length >= (dgrad ? 512 : 256) && tiles <= (dgrad && length < 1024 ? 128 : 256);
    return length >= 128 && tiles <= (length >= 1024 ? 768 : length >= 512 ? 512 : 256);
}
template <int FORM> bool takes_few(int T, int G, int K, int N, bool is16) {
    const int width = FORM == FWD ? N : K;
    return FORM != WGRAD && few_rows(likely_tiles(T, G, 32) * uem_cdiv(width, 32), FORM == FWD ? K : N, is16, FORM == DGRAD);
}
template <typename T, int FORM>
int launch_rows(const GgP& p, const char* what, hipStream_t st) {
    const int width = FORM == FWD ? p.N : p.K;
    if (takes_few<FORM>(p.T, p.G, p.K, p.N, sizeof(T) == 2)) {
        const int64_t items = (p.T / 32 + (int64_t)(p.G < p.T ? p.G : p.T)) * uem_cdiv(width, 32);
        constexpr int LDS = 16 * 32 * 36 * 4;
        if (uem_allow_lds((const void*)grouped_few_kernel<T, FORM>, LDS)) grouped_few_kernel<T, FORM><<<(unsigned)(uem_cdiv(items, 8) * 8), 1024, LDS, st>>>(p);
        return uem_check_launch(what);
    }
    const int t = pick_tile(p.T, p.G, width, sizeof(T) == 2);
    const int64_t items = (p.T / TILES[t].bm + (int64_t)(p.G < p.T ? p.G : p.T)) * uem_cdiv(width, TILES[t].bn);   // at most so many tiles: one of each group with rows is not full
    if (sizeof(T) == 2 && t == 0) return go<bf16_t, FORM, 256, 256, 2, 4>(p, items, what, st);
    if (t == 1) return go<T, FORM, 128, 128, 2, 2>(p, items, what, st);
    return go<T, FORM, 64, 128, 1, 4>(p, items, what, st);
}

template <int FORM>
int check(const void* a, const void* b, const void* out, const void* offsets, int T, int G, int K, int N, int lda, int ldb, int flags, const char* what) {
    const int es = (flags & UEM_GROUPED_BF16) ? 2 : 4;
    UEM_REQUIRE(a && b && out && offsets, "%s: null pointer", what);
    UEM_REQUIRE(T > 0 && G > 0 && K > 0 && N > 0 && T < (1 << 30) && G < (1 << 16) && K <= (1 << 20) && N <= (1 << 20),
                "%s: rows < 2^30, groups < 65536, K and N <= 2^20 (got %d, %d, %d, %d)", what, T, G, K, N);
    const uintptr_t at = (uintptr_t)a | (uintptr_t)b;
    if (takes_few<FORM>(T, G, K, N, es == 2)) UEM_REQUIRE(at % es == 0, "%s: operands must begin on element boundaries", what);
    else UEM_REQUIRE((at & 15) == 0 && (int64_t)lda * es % 16 == 0 && (int64_t)ldb * es % 16 == 0,
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
    const int per = (flags & UEM_GROUPED_BF16) ? 8 : 4;
    UEM_REQUIRE(src && dst && rows > 0 && cols > 0 && dst_ld >= cols && dst_ld % per == 0 && src_ld >= cols && ((uintptr_t)dst & 15) == 0,
                "grouped_pad: bad arguments (the copy's rows begin on 16-byte boundaries)");
    const int64_t chunks = rows * (dst_ld / per);
    const int grid = uem_stream_grid(chunks, 256);
    hipStream_t st = (hipStream_t)stream;
    if (per == 8) grouped_pad_kernel<bf16_t><<<grid, 256, 0, st>>>((const bf16_t*)src, src_ld, (bf16_t*)dst, dst_ld / per, cols, chunks);
    else grouped_pad_kernel<float><<<grid, 256, 0, st>>>((const float*)src, src_ld, (float*)dst, dst_ld / per, cols, chunks);
    return uem_check_launch("grouped_pad");
}
extern "C" int uem_grouped_any_rows(int T, int G, int K, int N, int flags, int dgrad) {
    const bool is16 = (flags & UEM_GROUPED_BF16) != 0;
    return dgrad ? takes_few<DGRAD>(T, G, K, N, is16) : takes_few<FWD>(T, G, K, N, is16);
}
extern "C" int uem_grouped_tile_rows(int T, int G, int K, int N, int flags, int form) {
    const bool is16 = (flags & UEM_GROUPED_BF16) != 0;
    UEM_REQUIRE(T > 0 && G > 0 && K > 0 && N > 0 && form >= FWD && form <= WGRAD, "grouped_tile_rows: bad arguments");
    if (form == WGRAD) return wgrad_tile(T, N, K, is16);
    if (form == FWD ? takes_few<FWD>(T, G, K, N, is16) : takes_few<DGRAD>(T, G, K, N, is16)) return 32;
    return TILES[pick_tile(T, G, form == FWD ? N : K, is16)].bm;
}
extern "C" int uem_grouped_fwd(const void* x, int x_ld, const void* w, int w_ld, const void* bias, void* y, const void* offsets, int T, int G, int K,
                               int N, int flags, void* stream) {
    const int rc = check<FWD>(x, w, y, offsets, T, G, K, N, x_ld, w_ld, flags, "grouped_fwd");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(x_ld >= K && w_ld >= K, "grouped_fwd: row strides shorter than the rows");
    GgP p = params(x, x_ld, w, w_ld, y, N, offsets, T, G, K, N, flags);
    p.bias = bias;
    return (flags & UEM_GROUPED_BF16) ? launch_rows<bf16_t, FWD>(p, "grouped_fwd", (hipStream_t)stream)
                                      : launch_rows<float, FWD>(p, "grouped_fwd", (hipStream_t)stream);
}
extern "C" int uem_grouped_dgrad(const void* dy, int dy_ld, const void* w, int w_ld, void* dx, const void* offsets, int T, int G, int K, int N, int flags,
                                 void* stream) {
    const int rc = check<DGRAD>(dy, w, dx, offsets, T, G, K, N, dy_ld, w_ld, flags, "grouped_dgrad");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(dy_ld >= N && w_ld >= K, "grouped_dgrad: row strides shorter than the rows");
    const GgP p = params(dy, dy_ld, w, w_ld, dx, K, offsets, T, G, K, N, flags);
    return (flags & UEM_GROUPED_BF16) ? launch_rows<bf16_t, DGRAD>(p, "grouped_dgrad", (hipStream_t)stream)
                                      : launch_rows<float, DGRAD>(p, "grouped_dgrad", (hipStream_t)stream);
}
extern "C" int64_t uem_grouped_wgrad_workspace_floats(int T, int G, int K, int N, int flags) {
    const int64_t slots = wgrad_slots(T, wgrad_chunk(T, G, N, K, wgrad_tile(T, N, K, (flags & UEM_GROUPED_BF16) != 0)));
    return (slots * (int64_t)N * K + 3) / 4 * 4 + slots * N;
}
extern "C" int uem_grouped_wgrad(const void* dy, int dy_ld, const void* x, int x_ld, void* dw, void* db, float* workspace, const void* offsets, int T,
                                 int G, int K, int N, int flags, void* stream) {
    const int rc = check<WGRAD>(dy, x, dw, offsets, T, G, K, N, dy_ld, x_ld, flags, "grouped_wgrad");
    if (rc != UEM_OK) return rc;
    UEM_REQUIRE(dy_ld >= N && x_ld >= K, "grouped_wgrad: row strides shorter than the rows");
    hipStream_t st = (hipStream_t)stream;
    GgP p = params(dy, dy_ld, x, x_ld, dw, K, offsets, T, G, K, N, flags);
    const bool h = (flags & UEM_GROUPED_BF16) != 0;
    const int bm = wgrad_tile(T, N, K, h);
    p.chunk = wgrad_chunk(T, G, N, K, bm);
    const int64_t slots = wgrad_slots(T, p.chunk), items = (T / p.chunk + (int64_t)G) * uem_cdiv(N, bm) * uem_cdiv(K, bm);
    UEM_REQUIRE(slots == 0 || (workspace && ((uintptr_t)workspace & 15) == 0), "grouped_wgrad: no workspace, or not on a 16-byte boundary");
    p.db = db;
    p.part = workspace;
    p.part_db = workspace + (slots * (int64_t)N * K + 3) / 4 * 4;
    const char* const what = "grouped_wgrad";
    const int launched = bm == 256 ? go<bf16_t, WGRAD, 256, 256, 2, 4>(p, items, what, st)
                         : h       ? go<bf16_t, WGRAD, 128, 128, 2, 2>(p, items, what, st)
                                   : go<float, WGRAD, 128, 128, 2, 2>(p, items, what, st);
    if (launched != UEM_OK) return launched;
    if (slots > 0) {
        const int64_t chunks = uem_cdiv(T, p.chunk), nb = uem_cdiv((int64_t)N * K, chunks > 64 ? 64 : chunks > 16 ? 256 : 1024);
        const int64_t most = slots / 2 < G ? slots / 2 : G;                    // groups of several chunks
        grouped_join_kernel<<<dim3((unsigned)(nb < 512 ? nb : 512) + 1, (unsigned)most), 256, 0, st>>>(p);
    }
    return uem_check_launch("grouped_wgrad");
}
