// Differential attention for gfx950, bf16 in / f32 accumulate, forward and gradient.
//
// A head has TWO softmax maps over 64-wide queries / keys and one 128-wide value (a head row is q1|q2, k1|k2, v: 128 columns each):
//     S_m = scale * Q_m K_m^T,   P_m = softmax over the row's visible keys,   lam = exp(l0.l1) - exp(l2.l3) + lam_init,
//     O = (P1 - lam P2) V,       Y = out_scale * gamma * O / sqrt(mean(O^2) + eps)      (Y = O without gamma).
// Query rows of the G = H / Hkv heads that share a key head are ONE list of R = G * Nq rows (row i * G + g: limits grow along it): shared key
// heads cost nothing extra in any pass and their gradients are summed inside a block, in a fixed order.
// Every mask here is a prefix: row i of clip b sees keys j < lim(b, i), lim = kv_len[b], cut at i + 1 (causal from the start) or at
// kv_len[b] - Nq + i + 1 (causal towards the end, new tokens behind a cache).  lim = 0: the row's outputs and gradients are zero.
// Rows of k / v at and behind kv_len[b] are never used: they are replaced by zeros on the way into LDS, whatever they hold.
//
// As in attention.hip, the first product is formed with the "other" sequence index on the LANE (v_mfma_f32_32x32x16_bf16):
//   forward / dQ : S^T[key][row] = K . Q^T, row softmax in-lane + one half swap;      dK, dV : S[row][key] = Q . K^T
// so the accumulator, packed to bf16, is the B operand of the second product.  Softmax sums, statistics, lambda and norms stay in f32.
// Rounded to bf16 between the inputs and the results, each by half a step at most (2^-8 of the value; 1.7e-3 in the 2-norm):
//   P (forward), A = P1 - lam P2 and dS (gradient), dO behind the norm: operands of matrix products, which take bf16 -- two terms each would
//   be twice the products;
//   the saved o and o2, from which the gradient forms the norm and dO . O1, dO . O2 again: f32 ones would be 512 bytes more a
//   head row to write and as many to read, by the bytes 30 us at 32 x 1568 x 3 heads, and take 0.7e-3, in squares, off dq and dk.
// 2-norms against 64 bits (32 x 160 x 6 heads): outputs 2.2e-3, dv 3.1e-3, dq and dk 3.6e-3; a rounding of the exact results alone is 1.7e-3.
#include "common.h"
#include "../../include/mofo_hip.h"
#include <algorithm>
#include <type_traits>

namespace {

#include "attn_tile.h"

constexpr int HV = 128;                 // columns of a head's q, k, v and output rows
constexpr float EMPTY_LSE = 1.0e30f;    // log-sum of a row that sees nothing: exp2(s - 1e30) = 0
// Forward: a row's reference maximum is kept until a score lies more than this many log2 units above it.  The row's outputs are divided
// by the sum of the ROUNDED terms, so that the rounding of a term that dominates its row cancels; the reference follows a term that is
// far above it, which is then 1 and not rounded at all.  (Gradients are formed from differences G - d in which such a term cancels: with
// the sum of the unrounded terms and a reference kept up to 2^20, dq of 160 and 50 tokens was 6e-3 and 1e-2 off.  This way 3.6e-3 for 160
// tokens; kept up to 2^2.5 it is 3.0e-3, and the training step of 32 x 1568 x 3 heads 3 % longer, with the maximum always followed 2.7e-3.)
constexpr float KEEP_REF = 5.f;
// Exponents are c s - c (reference) in one fused step while a row's reference lies below this many log2 units: the rounding of c (reference),
// 2^-15, is the same for all of a row's terms of one reference, and that small against those of another.  Beyond it the reference is taken
// off the row's scores first, exactly; a wave with such a row looks at every tile's references.  A row's numbers are its own either way.
constexpr float FAR_REF = 1024.f;

struct DiffArgs {
    const bf16_t *q, *k, *v;
    size_t ldq, ldk, ldv;
    int B, H, Hkv, G, Nq, Nk, R, causal;
    int row0;                 // forward and dQ: the launch's first row of every list
    const int* kv_len;
    const void* lam;          // [4][lam_heads][64]
    const void* gamma;        // [128] or NULL
    int param_bf16, lam_heads;
    float lam_init, scale, c, eps, out_scale;
};

__device__ __forceinline__ int clip_len(const DiffArgs& a, int b) {
    if (!a.kv_len) return a.Nk;
    const int n = a.kv_len[b];
    return n < 0 ? 0 : n > a.Nk ? a.Nk : n;
}
// causal masks: row i sees the first i + past(len) keys at most
__device__ __forceinline__ int past(const DiffArgs& a, int len) { return a.causal == 0 ? 1 << 30 : a.causal == 1 ? 1 : len - a.Nq + 1; }
__device__ __forceinline__ int row_lim(const DiffArgs& a, int len, int i) { return max(0, min(len, i + past(a, len))); }
// smallest and largest limit of the rows ra .. rb (inclusive) of the list
__device__ __forceinline__ void span_lim(const DiffArgs& a, int len, int ra, int rb, int& lo, int& hi) {
    lo = row_lim(a, len, a.G == 1 ? ra : ra / a.G);
    hi = row_lim(a, len, a.G == 1 ? rb : rb / a.G);
}
__device__ __forceinline__ float param(const void* p, int bf, size_t i) { return bf ? bf16_to_f32(((const bf16_t*)p)[i]) : ((const float*)p)[i]; }
// sum over the wave, in every lane, by lane permutes inside the vector unit (a shuffle goes through LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_sum_dpp(float x) {
    x = dpp_add<0x111, 0xf>(x);      // row_shr 1, 2, 4, 8: lane 15 of every row of 16 holds the row's sum
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);      // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3: lane 63 holds all
    x = dpp_add<0x143, 0xc>(x);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
// lambda of head h, and its two exponentials (every lane of the wave)
__device__ __forceinline__ float head_lambda(const DiffArgs& a, int h, int lane, float& e1, float& e2) {
    const int hl = a.lam_heads == 1 ? 0 : h;
    const size_t st = (size_t)a.lam_heads * 64, o = (size_t)hl * 64 + lane;
    e1 = expf(wave_sum_dpp(param(a.lam, a.param_bf16, o) * param(a.lam, a.param_bf16, st + o)));
    e2 = expf(wave_sum_dpp(param(a.lam, a.param_bf16, 2 * st + o) * param(a.lam, a.param_bf16, 3 * st + o)));
    return e1 - e2 + a.lam_init;
}

__device__ __forceinline__ float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ f32x16 mfma(bf16x8 x, bf16x8 y, f32x16 acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0); }

// A lane's byte offsets into a [32][64] half tile, LDS base included (the base a multiple of 128): k step ks of the rows is row ^ 32 ks, columns
// 32 dt .. 32 dt + 31 are tr ^ 64 dt (first and second four rows of a k step); everything else about a fragment's address is a constant.
// RowOff / ColOff are made where a phase of a tile begins: kept through a tile loop they would be eight registers.
#define LDS_AS __attribute__((address_space(3)))
struct FragOff {
    unsigned row, tr0, tr1;
};
__device__ __forceinline__ FragOff frag_off(unsigned lds, int lane) {
    const int r = lane & 31, hh = lane >> 5, gg = lane >> 4, i = lane & 15, q = i >> 2, pp = i & 3, ra = 4 * hh + q, rb = ra + 8;
    const int chunk = 2 * (gg & 1) + (pp >> 1), sub = (pp & 1) * 8;
    return {lds + r * RS + ((hh ^ swz(r)) << 4), lds + ra * RS + ((chunk ^ swz(ra)) << 4) + sub, lds + rb * RS + ((chunk ^ swz(rb)) << 4) + sub};
}
struct RowOff {
    unsigned o[4];
    __device__ __forceinline__ RowOff(const FragOff& f, unsigned base = 0) {
        unsigned x = f.row + base;
        asm volatile("" : "+v"(x));
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) o[ks] = x ^ (32 * ks);
    }
    __device__ __forceinline__ bf16x8 get(unsigned tile, int ks) const { return *(const LDS_AS bf16x8*)(size_t)(o[ks] + tile); }     // as row_frag
};
struct ColOff {
    unsigned o[2][2];
    __device__ __forceinline__ ColOff(const FragOff& f, unsigned base = 0) {
        unsigned x = f.tr0 + base, y = f.tr1 + base;
        asm volatile("" : "+v"(x), "+v"(y));
        o[0][0] = x;
        o[0][1] = y;
        o[1][0] = x ^ 64;
        o[1][1] = y ^ 64;
    }
    __device__ __forceinline__ bf16x8 get(unsigned tile, int s2, int dt) const {                                                       // as tr_frag
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(size_t)(o[dt][0] + tile + 16 * RS * s2));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(size_t)(o[dt][1] + tile + 16 * RS * s2));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        return __builtin_bit_cast(bf16x8, u32x4{l2[0], l2[1], h2[0], h2[1]});
    }
};

// Blocks are dealt round-robin over the 8 XCDs, each with an L2 of its own.  Mostly: the blocks of one (clip, key head) next to each other,
// every XCD an eighth of that list, so that K and V are fetched by one XCD or two.  `spread`: over all XCDs, the longest blocks of all
// heads first -- few heads, causal or of ragged lengths, where eighths of the list would be far from equal.  Causal blocks differ in
// length along x (long ones at the end: `late`, or at the start): within an eighth long and short ones alternate along the list, and the
// long ones start first.
__device__ __forceinline__ bool place_block(const DiffArgs& a, int id, int nx, int spread, bool late, int& x, int& b, int& kvh) {
    const int groups = a.B * a.Hkv, n = groups * nx;
    int g, q;
    if (spread) {
        if (id >= n) return false;
        q = id / groups;
        g = id - q * groups;
        x = a.causal && late ? nx - 1 - q : q;
    } else {
        const int per = (n + 7) >> 3, lo = (id & 7) * per, have = min(per, n - lo), j = id >> 3;
        if (j >= have) return false;
        const int half = (have + 1) >> 1, pos = lo + (!a.causal ? j : j < half ? 2 * j : 2 * (have >> 1) - 1 - 2 * (j - half));
        g = pos / nx;
        q = pos - g * nx;
        x = !a.causal ? q : (q & 1) ? q >> 1 : nx - 1 - (q >> 1);
        if (a.causal && !late) x = nx - 1 - x;
    }
    b = g / a.Hkv;
    kvh = g - b * a.Hkv;
    return true;
}

// one lane's row of a wave tile
struct Row {
    bool valid;
    int h, i, lim;
};
__device__ __forceinline__ size_t row_at(const DiffArgs& a, int b, const Row& w) { return (size_t)b * a.Nq + w.i; }                       // of q, out, dout
__device__ __forceinline__ size_t stat_at(const DiffArgs& a, int b, const Row& w) { return ((size_t)b * a.H + w.h) * a.Nq + w.i; }    // of [B, H, Nq]
__device__ __forceinline__ Row make_row(const DiffArgs& a, int kvh, int r, int len) {
    Row w;
    w.valid = r < a.R;
    if (!w.valid) r = a.R - 1;
    w.i = a.G == 1 ? r : r / a.G;
    w.h = kvh * a.G + r - w.i * a.G;
    w.lim = w.valid ? row_lim(a, len, w.i) : 0;
    return w;
}

// A wave's 32 rows of 128 results, held in accumulator layout (row on the lane), leave through its own piece of LDS as whole rows: 16 bytes a
// lane, 256 bytes a row (straight from the accumulators a store covers 16 bytes of each of 32 rows, 2.1 TB/s).
constexpr int OUT_ROW = 272, OUT_WAVE = 32 * OUT_ROW;       // rows padded by 16 bytes: no bank conflicts
__device__ __forceinline__ void out_put(unsigned char* lds, int lane, int dt, int rg, float v0, float v1, float v2, float v3) {
    *(u32x2*)(lds + (lane & 31) * OUT_ROW + 64 * dt + 16 * rg + 8 * (lane >> 5)) = u32x2{pack_bf16x2(v0, v1), pack_bf16x2(v2, v3)};
}
__device__ __forceinline__ void out_put16(unsigned char* lds, int lane, int dt, const f32x16& x, float mul) {
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) out_put(lds, lane, dt, rg, x[4 * rg] * mul, x[4 * rg + 1] * mul, x[4 * rg + 2] * mul, x[4 * rg + 3] * mul);
}
// row(r): where row r of the tile goes, or NULL
template <class F>
__device__ __forceinline__ void out_flush(const unsigned char* lds, int lane, F row, int j0 = 0, int j1 = 8) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = j0; j < j1; ++j) {
        const int r = 4 * j + (lane >> 4);
        const u32x4 x = *(const u32x4*)(lds + r * OUT_ROW + (lane & 15) * 16);
        bf16_t* p = row(r);
        if (p) *(u32x4*)(p + (lane & 15) * 8) = x;
    }
    __builtin_amdgcn_wave_barrier();
}
// row r0 + r of the list in a tensor of row pitch ld, columns of its head
__device__ __forceinline__ bf16_t* list_row(const DiffArgs& a, bf16_t* base, size_t ld, int b, int kvh, int r) {
    if (r >= a.R) return nullptr;
    const int i = a.G == 1 ? r : r / a.G;
    return base + ((size_t)b * a.Nq + i) * ld + (size_t)(kvh * a.G + r - i * a.G) * HV;
}

// LDS-DMA of one operand's [32 rows][64 columns] half tile, as four pieces of 8 rows; rows that are not there come from a line of zeros
__device__ const u32x4 g_zero = {0, 0, 0, 0};
struct HalfTile {
    const bf16_t* base;     // first row's 64 columns
    size_t ld;
    int voff[2];            // byte offset of the lane's 16 bytes inside the first / second piece of 8 rows (the swizzle sits on the source column)
};
__device__ __forceinline__ HalfTile half_tile(const bf16_t* base, size_t ld, int lane) {
    HalfTile t;
    t.base = base;
    t.ld = ld;
#pragma unroll
    for (int o = 0; o < 2; ++o) t.voff[o] = (int)(((size_t)(8 * o + (lane >> 3)) * ld + (((lane & 7) ^ swz(8 * o + (lane >> 3))) << 3)) * 2);
    return t;
}
// Four pieces, 1 KiB each; the third and fourth lie 16 rows (p1) behind the first two.  One block: a scalar base that a vector instruction
// wrote may be read five states later, M0 one state after it is written.
__device__ __forceinline__ void dma_pieces(const void* p0, const void* p1, int v0, int v1, unsigned lds_dst) {
    unsigned keep;
    asm volatile(
        "s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\t"
        "s_add_u32 m0, %5, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %1\n\t"
        "s_add_u32 m0, %5, 0x800\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\t"
        "s_add_u32 m0, %5, 0xc00\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %2\n\ts_mov_b32 m0, %0"
        : "=&s"(keep)
        : "s"(p0), "s"(p1), "v"(v0), "v"(v1), "s"(lds_dst)
        : "memory", "scc");
}
// rows in front of `first` and at and behind `rows` are zero
__device__ __forceinline__ void dma_edge(const HalfTile& t, int row0, int rows, unsigned lds_dst, int lane, int first) {
    asm volatile("" : "+v"(lane));         // nothing of this path is to be kept in registers across a tile loop
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
        const int rl = 8 * sub + (lane >> 3), row = row0 + rl;
        const void* src = row >= first && row < rows ? (const void*)(t.base + (size_t)row * t.ld + (((lane & 7) ^ swz(rl)) << 3)) : (const void*)&g_zero;
        dma_b128(src, lds_dst + sub * 1024);
    }
}
__device__ __forceinline__ void dma_inside(const HalfTile& t, int row0, unsigned lds_dst) {
    const bf16_t* p = t.base + (size_t)row0 * t.ld;
    dma_pieces(p, p + t.ld * 16, t.voff[0], t.voff[1], lds_dst);
}
__device__ __forceinline__ void dma_half_tile(const HalfTile& t, int row0, int rows, unsigned lds_dst, int lane, int first = 0) {
    if (row0 >= first && row0 + 32 <= rows) dma_inside(t, row0, lds_dst);
    else dma_edge(t, row0, rows, lds_dst, lane, first);
}
// both halves of a 128-wide row, of two tensors: four half tiles
__device__ __forceinline__ void dma_tiles(HalfTile x, HalfTile y, int row0, int rows, unsigned lds_dst, int lane, int first = 0) {
    HalfTile x1 = x, y1 = y;
    x1.base += 64;
    y1.base += 64;
    if (row0 >= first && row0 + 32 <= rows) {
        dma_inside(x, row0, lds_dst);
        dma_inside(x1, row0, lds_dst + TILE);
        dma_inside(y, row0, lds_dst + 2 * TILE);
        dma_inside(y1, row0, lds_dst + 3 * TILE);
    } else {
        dma_edge(x, row0, rows, lds_dst, lane, first);
        dma_edge(x1, row0, rows, lds_dst + TILE, lane, first);
        dma_edge(y, row0, rows, lds_dst + 2 * TILE, lane, first);
        dma_edge(y1, row0, rows, lds_dst + 3 * TILE, lane, first);
    }
}
// own pieces but the N newest have landed, own LDS reads are done; then every wave's
template <int N>
__device__ __forceinline__ void landed_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// KEYS4 blocks (few rows, or few blocks): four waves share 32 rows and deal the key tiles -- or a wave's 32 keys the row tiles -- among
// themselves.  Every wave has one tile of its own, refilled when its last read is done (two such blocks on a compute unit cover each
// other's waits), and meets the others only at the end, where the four sums are added up through LDS in a fixed order.
__device__ __forceinline__ void landed_own() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void acc_put(unsigned char* lds, int unit, int lane, const f32x16& x, float mul) {
#pragma unroll
    for (int rg = 0; rg < 4; ++rg)
        *(f32x4*)(lds + unit * 4096 + rg * 1024 + lane * 16) = f32x4{x[4 * rg] * mul, x[4 * rg + 1] * mul, x[4 * rg + 2] * mul, x[4 * rg + 3] * mul};
}
// sum over the four waves of one accumulator: wave v's unit lies at v * stride + unit * 4096
__device__ __forceinline__ f32x16 acc_sum(const unsigned char* lds, int stride, int unit, int lane) {
    f32x16 x;
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
        f32x4 t = *(const f32x4*)(lds + unit * 4096 + rg * 1024 + lane * 16);
#pragma unroll
        for (int v = 1; v < 4; ++v) t += *(const f32x4*)(lds + v * stride + unit * 4096 + rg * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * rg + e] = t[e];
    }
    return x;
}

// a four-way wave's LDS reads are done: its one tile may be overwritten
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ------------------------------------------------------------------------------------------------ forward
struct FwdOut {
    bf16_t *out, *o, *o2;     // out [B * Nq, ldo]; o, o2 [B * Nq, H * 128] or NULL
    size_t ldo;
    float* lse2;              // [2][B][H][Nq] or NULL
    float* part;              // nsplit > 1: [rows][nsplit][2][128] outputs of a range of keys, divided by its own sum, then
    f32x2* part_stat;         // [rows][nsplit][2] its reference (score units) and its log2-sum against it (both -inf: nothing seen); rows = B * H * Nq
};

// sum of the eight rounded terms of a fragment
__device__ __forceinline__ float frag_sum(bf16x8 f, float acc) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    const u32x4 w = __builtin_bit_cast(u32x4, f);
    const bf16x2 one = __builtin_bit_cast(bf16x2, 0x3f803f80u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t pair = w[e];       // (a bit cast of the vector's element itself reads element 0)
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), one, acc, false);
    }
    return acc;
}

// One block: four waves of 32 rows that share the key tiles of one (clip, key head), two tiles a barrier in a ring of four filled by LDS-DMA;
// or KEYS4.  nsplit > 1: of a range of the keys, joined by diff_join_kernel.
// 24 matrix instructions (768 cycles of the matrix unit) and about 150 others, 32 of them exponentials at twice the time (740 cycles), stand
// against the 1850 cycles a tile that a SIMD takes: matrix unit 39 % and vector unit 45 % busy, LDS 15 %, two waves a SIMD (the
// registers allow no third) whose phases meet too often, at the 1.9 to 2.1 GHz that the card holds.  16 clips x 6 heads x 1568 tokens
// 211 us, 573 TFLOP/s; one clip of 12544 752 to 762 us, 640 TFLOP/s; one clip of 1568 29 us.  (FLOP as the formula has them, 512 a row and key; each
// map's own second product makes 768 of it, since neither sum is known before the last key: 16 x 6 x 2048, whose blocks fill three rounds,
// runs at 620 to 664, that is up to 996 TFLOP/s of matrix work, 83 % of a large library product's rate.)  At 1568, without exponentials it is 7 % faster,
// without the second products 23 %, without loads 10 %.  Tried without gain: blocks of eight waves whose two halves do products and
// softmax in opposite phases, a barrier between; the two maps' first products in turn; the next tile's first fragments ahead of the
// barrier; fences that interleave exponentials and products.  One wave a SIMD, a tile ahead, needs copies between the two halves of the
// register file.
template <bool KEYS4, bool SAVE, bool SPLIT>
__global__ __launch_bounds__(256, 2) void diff_fwd_kernel(DiffArgs a, FwdOut f, int nx, int nsplit, int spread) {
    constexpr int STAGE = 4 * TILE, ROWS = KEYS4 ? 32 : 128, XCH = 4 * STAGE;
    __shared__ __attribute__((aligned(128))) unsigned char smem[XCH + (KEYS4 ? 4096 : 0)];
    __shared__ float gam[HV], lams[KEYS4 ? 32 : 1];         // KEYS4: the rows' lambda, out of the registers during the loop
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int xs, b, kvh;
    if (!place_block(a, blockIdx.x, nx * nsplit, spread, true, xs, b, kvh)) return;
    const int xb = xs / nsplit, sp = xs - xb * nsplit;
    const int len = clip_len(a, b);
    const int rb0 = a.row0 + xb * ROWS, r0 = rb0 + (KEYS4 ? 0 : wave * 32);
    const Row w = make_row(a, kvh, r0 + (lane & 31), len);
    int wlo = 0, whi = 0, blo, bhi;
    span_lim(a, len, rb0, min(rb0 + ROWS, a.R) - 1, blo, bhi);
    if (r0 < a.R) span_lim(a, len, r0, min(r0 + 32, a.R) - 1, wlo, whi);
    // this block's range of key tiles; KEYS4: the wave's own are t0 + wave, t0 + wave + 4, ...
    const int tiles = (bhi + 31) >> 5, chunk = ((a.Nk + 31) / 32 + nsplit - 1) / nsplit;
    const int t0 = min(sp * chunk, tiles), t1 = min(t0 + chunk, tiles), all = t1 - t0;
    const int first = KEYS4 ? t0 + wave : t0, stride = KEYS4 ? 4 : 1, nkt = KEYS4 ? (all - wave + 3) >> 2 : all;

    const bf16_t* kp = a.k + (size_t)b * a.Nk * a.ldk + (size_t)kvh * HV;
    const bf16_t* vp = a.v + (size_t)b * a.Nk * a.ldv + (size_t)kvh * HV;
    HalfTile ht = half_tile((KEYS4 || wave < 2 ? kp : vp) + (KEYS4 ? 0 : (wave & 1) * 64), KEYS4 || wave < 2 ? a.ldk : a.ldv, lane), hv;
    if constexpr (KEYS4) hv = half_tile(vp, a.ldv, lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem), ring = KEYS4 ? wave * STAGE : 0;
    auto issue = [&](int t, unsigned buf) {
        const int row0 = (first + t * stride) * 32;
        const unsigned at = lds0 + ring + buf * STAGE;
        if constexpr (KEYS4) {
            dma_tiles(ht, hv, row0, len, at, lane);
        } else {
            dma_half_tile(ht, row0, len, at + wave * TILE, lane);
        }
    };
    if (nkt > 0) issue(0, 0);
    if (!KEYS4 && nkt > 1) issue(1, 1);

    bf16x8 qf[2][4];
    const bf16_t* qp = a.q + row_at(a, b, w) * a.ldq + (size_t)w.h * HV;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[m][ks] = *(const bf16x8*)(qp + 64 * m + 16 * ks + 8 * hh);

    // the epilogue's numbers, while the first tiles are on their way: the heads' lambda, gamma times out_scale
    float lam = 0.f;
    if constexpr (!SPLIT) {
        float e1, e2;
        for (int h = kvh * a.G; h < (kvh + 1) * a.G; ++h) {
            const float t = head_lambda(a, h, lane, e1, e2);
            lam = w.h == h ? t : lam;
        }
        if (KEYS4 && tid < 32) lams[tid] = lam;
        if (a.gamma && tid < HV) gam[tid] = a.out_scale * param(a.gamma, a.param_bf16, tid);
    }

    f32x16 o[2][4];
    float mx[2], l[2], le[2];          // reference maximum, sum of the rounded terms, sum of the unrounded terms (SAVE)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        mx[m] = -__builtin_inff();
        l[m] = le[m] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[m][dt] = zero16();
    }

    const FragOff fo = frag_off(lds0 + ring, lane);
    const float keep = uniform(KEEP_REF / a.c);           // in score units
    float look = keep;                                    // -inf once a row's reference is far: every tile takes the branch below
    auto is_far = [&](float x) { return x > -__builtin_inff() && fabsf(x * a.c) > FAR_REF; };
    for (int t = 0; t < nkt; ++t) {
        if constexpr (KEYS4) {
            landed_own();
        } else if ((t & 1) == 0) {
            landed_barrier<0>();
            if (t + 2 < nkt) issue(t + 2, (t + 2) & 3);
            if (t + 3 < nkt) issue(t + 3, (t + 3) & 3);
        }
        const unsigned buf = KEYS4 ? 0 : t & 3;
        const int k0 = (first + t * stride) * 32;
        const unsigned T = buf * STAGE;
        if (k0 >= whi) continue;                          // no row of this wave sees the tile (KEYS4: one does)
        // fragment registers are refilled right behind the matrix instruction that read them
        bf16x8 fr[4];
        RowOff ro(fo, T);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) fr[ks] = ro.get(0, ks);
        f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            s[0] = mfma(fr[ks], qf[0][ks], s[0]);
            fr[ks] = ro.get(TILE, ks);
        }
        ColOff co(fo, T);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            s[1] = mfma(fr[ks], qf[1][ks], s[1]);
            fr[ks] = co.get((2 + (ks >> 1)) * TILE, 0, ks & 1);
        }
        if (k0 + 32 > wlo) {
            int lim = w.lim - k0 - 4 * hh;
            asm volatile("" : "+v"(lim));
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((r & 3) + 8 * (r >> 2) >= lim) s[0][r] = s[1][r] = -__builtin_inff();
        }
        float tm[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            tm[m] = s[m][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) tm[m] = fmaxf(tm[m], s[m][r]);
            if (m == 0) __builtin_amdgcn_sched_barrier(0);      // the first map's maximum while the second's scores are on their way
        }
        float taken[2] = {0.f, 0.f};                      // what the scores are already less by
        if (__any(!(tm[0] <= mx[0] + look) || !(tm[1] <= mx[1] + look))) {    // the first tile (reference -inf) too
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float x = fmaxf(tm[m], __shfl_xor(tm[m], 32, 64));
                const bool up = x > mx[m] + keep;
                const float alpha = up ? fast_exp2((mx[m] - x) * a.c) : 1.f;
                mx[m] = up ? x : mx[m];
                l[m] *= alpha;
                if constexpr (SAVE) le[m] *= alpha;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[m][dt][r] *= alpha;
            }
            const bool far[2] = {is_far(mx[0]), is_far(mx[1])};
            if (__ballot(far[0] || far[1]) != 0) {
                look = -__builtin_inff();
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    taken[m] = far[m] ? mx[m] : 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[m][r] -= taken[m];
                }
            }
        }
        // two halves of 16 keys: the second half's exponentials stand beside the first half's products
        const float nmc[2] = {(taken[0] - mx[0]) * a.c, (taken[1] - mx[1]) * a.c};
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            if (KEYS4 && s2 == 1) {
                reads_done();
                if (t + 1 < nkt) issue(t + 1, 0);
            }
            bf16x8 pf[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    p[r] = fast_exp2(fmaf(s[m][8 * s2 + r], a.c, nmc[m]));
                    if constexpr (SAVE) le[m] += p[r];
                }
                pf[m] = pack_frag(p, 0);
                l[m] = frag_sum(pf[m], l[m]);
            }
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                o[0][dt] = mfma(fr[dt], pf[0], o[0][dt]);
                o[1][dt] = mfma(fr[dt], pf[1], o[1][dt]);
                if (s2 == 0) fr[dt] = co.get((2 + (dt >> 1)) * TILE, 1, dt & 1);
            }
        }
    }

    bool some = w.lim > first * 32 && nkt > 0;             // the row sees a key of this wave's
    float lt[2], lx[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        lt[m] = l[m] + __shfl_xor(l[m], 32, 64);
        lx[m] = SAVE ? le[m] + __shfl_xor(le[m], 32, 64) : lt[m];
    }
    float inv[2];
    // a row's statistics leave as soon as they are known: the map's reference (score units) and the sum of its terms against that
    int row_lane = lane & 31;
    asm volatile("" : "+v"(row_lane));                    // the row's place is made anew: kept through the loop it would not fit the registers
    const Row at = make_row(a, kvh, r0 + row_lane, len);
    auto put_stat = [&](int m, bool seen, float ref, float sum) {
        if (!at.valid || hh != 0 || (KEYS4 && wave != 0)) return;
        if constexpr (SPLIT) f.part_stat[(stat_at(a, b, at) * nsplit + sp) * 2 + m] = seen ? f32x2{ref, fast_log2(sum)} : f32x2{-__builtin_inff(), -__builtin_inff()};
        else if constexpr (SAVE) f.lse2[(size_t)m * a.B * a.H * a.Nq + stat_at(a, b, at)] = seen ? ref * a.c + fast_log2(sum) : EMPTY_LSE;
    };
    float* xch = (float*)(smem + XCH);
    if constexpr (KEYS4) {
        // the four waves' references and sums, [wave][map][reference, rounded sum, sum][32 rows]; a wave without keys of the row: nothing
        __syncthreads();
        if (hh == 0) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float* p = xch + (wave * 2 + m) * 96 + lane;
                p[0] = some ? mx[m] : -__builtin_inff();
                p[32] = some ? lt[m] : 0.f;
                p[64] = some ? lx[m] : 0.f;
            }
        }
        __syncthreads();
        const bool any = w.lim > t0 * 32 && all > 0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float top = -__builtin_inff(), st = 0.f, sx = 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float x = xch[(v * 2 + m) * 96 + (lane & 31)];
                top = x > top ? x : top;
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float* p = xch + (v * 2 + m) * 96 + (lane & 31);
                const float e = p[32] != 0.f ? fast_exp2((p[0] - top) * a.c) : 0.f;
                st += e * p[32];
                sx += e * p[64];
            }
            inv[m] = some ? fast_exp2((mx[m] - top) * a.c) / st : 0.f;
            put_stat(m, any, top, sx);
        }
        // a map at a time (there is no room for both); wave w goes on with columns 32 w .. 32 w + 31
        f32x16 sum[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                int on = some;                            // opaque: the selects of all eight tiles at once do not fit the registers
                asm volatile("" : "+v"(on));
                f32x16 x = o[m][dt];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = on ? x[r] : 0.f;           // whatever a row that sees nothing holds
                acc_put(smem + wave * STAGE, dt, lane, x, inv[m]);
            }
            __syncthreads();
            sum[m] = acc_sum(smem, STAGE, wave, lane);
            if (m == 0) __syncthreads();
        }
        some = any;
        lam = lams[lane & 31];
        o[0][0] = sum[0];
        o[1][0] = sum[1];
        inv[0] = inv[1] = 1.f;
    } else {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            inv[m] = some ? 1.0f / lt[m] : 0.f;
            put_stat(m, some, mx[m], lx[m]);
        }
    }
    constexpr int ND = KEYS4 ? 1 : 4;                     // column tiles this wave still holds, from dt0 on
    const int dt0 = KEYS4 ? wave : 0;
    if constexpr (SPLIT) {
        if (!at.valid || all <= 0) return;                // the join does not use a range of weight zero
        float* pp = f.part + (stat_at(a, b, at) * nsplit + sp) * (2 * HV);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int rg = 0; rg < 4; ++rg) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = some ? o[m][dt][4 * rg + e] * inv[m] : 0.f;
                    *(f32x4*)(pp + m * HV + 32 * (dt0 + dt) + 8 * rg + 4 * hh) = x;
                }
        }
    } else {
    __syncthreads();                                      // the ring is free, the sums are read
    // KEYS4: the waves' columns meet in one tile (per output) and leave it 8 rows a wave
    unsigned char* lds = smem + (KEYS4 ? 0 : wave * OUT_WAVE);
    constexpr int NEXT = KEYS4 ? OUT_WAVE : 0;            // o2, o, out: one place after the other, or three
    float ss = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = some ? o[1][dt][4 * rg + e] * inv[1] : 0.f;
                x[e] = some ? fmaf(-lam, y[e], o[0][dt][4 * rg + e] * inv[0]) : 0.f;
                ss = fmaf(x[e], x[e], ss);
                o[0][dt][4 * rg + e] = x[e];
            }
            if constexpr (SAVE) out_put(lds, lane, dt0 + dt, rg, y[0], y[1], y[2], y[3]);
        }
        __builtin_amdgcn_sched_barrier(0);                // everything at once does not fit beside the accumulators
    }
    const size_t HW = (size_t)a.H * HV;
    if constexpr (SAVE) {
        if (!KEYS4) out_flush(lds, lane, [&](int r) { return list_row(a, f.o2, HW, b, kvh, r0 + r); });
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) out_put16(lds + NEXT, lane, dt0 + dt, o[0][dt], 1.f);
        if (!KEYS4) out_flush(lds, lane, [&](int r) { return list_row(a, f.o, HW, b, kvh, r0 + r); });
    }
    if (a.gamma) {
        ss += __shfl_xor(ss, 32, 64);
        if constexpr (KEYS4) {
            if (hh == 0) xch[wave * 32 + lane] = ss;
            __syncthreads();
            ss = (xch[lane & 31] + xch[32 + (lane & 31)]) + (xch[64 + (lane & 31)] + xch[96 + (lane & 31)]);
        }
        const float rn = 1.0f / sqrtf(ss * (1.f / HV) + a.eps);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
#pragma unroll
            for (int rg = 0; rg < 4; ++rg) {
                const f32x4 gm = *(const f32x4*)(gam + 32 * (dt0 + dt) + 8 * rg + 4 * hh);
                out_put(lds + 2 * NEXT, lane, dt0 + dt, rg, o[0][dt][4 * rg] * rn * gm[0], o[0][dt][4 * rg + 1] * rn * gm[1], o[0][dt][4 * rg + 2] * rn * gm[2],
                        o[0][dt][4 * rg + 3] * rn * gm[3]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    } else if (!SAVE || KEYS4) {
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) out_put16(lds + 2 * NEXT, lane, dt0 + dt, o[0][dt], 1.f);
    }
    if constexpr (KEYS4) {
        __syncthreads();
        if constexpr (SAVE) {
            out_flush(lds, lane, [&](int r) { return list_row(a, f.o2, HW, b, kvh, r0 + r); }, 2 * wave, 2 * wave + 2);
            out_flush(lds + NEXT, lane, [&](int r) { return list_row(a, f.o, HW, b, kvh, r0 + r); }, 2 * wave, 2 * wave + 2);
        }
        out_flush(lds + 2 * NEXT, lane, [&](int r) { return list_row(a, f.out, f.ldo, b, kvh, r0 + r); }, 2 * wave, 2 * wave + 2);
    } else {
        out_flush(lds, lane, [&](int r) { return list_row(a, f.out, f.ldo, b, kvh, r0 + r); });
    }
    }
}

// joins the ranges of a row: one wave a row, lanes 0..31 the first map's 128 columns, lanes 32..63 the second's; the ranges' weights are
// exp2(c (reference - largest reference) + log2-sum) over their sum, lane s of a half holding ranges s and s + 32.  A chain of latencies: the
// first sixteen ranges' loads go out before anything is waited for (one token against 16 caches of 8192, 16 ranges: 5.7 us, 6.5 in rounds of eight behind the weights).
__global__ __launch_bounds__(256) void diff_join_kernel(DiffArgs a, FwdOut f, int nsplit) {
    constexpr int AT_ONCE = 16;
    const int lane = threadIdx.x & 63, m = lane >> 5, sl = lane & 31, d = sl * 4;
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (size_t)a.B * a.H * a.Nq;
    if (row >= rows) return;
    const f32x2* pl = f.part_stat + row * nsplit * 2 + m;
    const f32x2 nothing = {-__builtin_inff(), -__builtin_inff()};
    const f32x2 v0 = sl < nsplit ? pl[2 * sl] : nothing, v1 = sl + 32 < nsplit ? pl[2 * (sl + 32)] : nothing;
    const float* pp = f.part + row * nsplit * (2 * HV) + m * HV + d;
    f32x4 x[AT_ONCE];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) x[j] = *(const f32x4*)(pp + (size_t)min(s0 + j, nsplit - 1) * (2 * HV));
    };
    fetch(0);
    const size_t bh = row / a.Nq;
    const int i = (int)(row - bh * a.Nq), b = (int)(bh / a.H), h = (int)(bh - (size_t)b * a.H);
    f32x4 gam = {1.f, 1.f, 1.f, 1.f};
    if (a.gamma) {
#pragma unroll
        for (int e = 0; e < 4; ++e) gam[e] = param(a.gamma, a.param_bf16, d + e);
    }
    float e1, e2;
    const float lam = head_lambda(a, h, lane, e1, e2);
    float top = fmaxf(v0[0], v1[0]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    // a NaN among a range's scores leaves its log-sum NaN, and makes the row NaN
    const bool none = (uint32_t)(__ballot(v0[1] != -__builtin_inff() || v1[1] != -__builtin_inff()) >> (lane & 32)) == 0;
    float w0 = none ? 0.f : fast_exp2(fmaf(v0[0] - top, a.c, v0[1])), w1 = none ? 0.f : fast_exp2(fmaf(v1[0] - top, a.c, v1[1])), sum = w0 + w1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float lse = none ? EMPTY_LSE : top * a.c + fast_log2(sum), inv = none ? 0.f : 1.0f / sum;
    w0 *= inv;
    w1 *= inv;
    f32x4 acc = {0, 0, 0, 0};
    for (int s0 = 0; s0 < nsplit; s0 += AT_ONCE) {
        if (s0) fetch(s0);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const float w = __shfl(s0 < 32 ? w0 : w1, (lane & 32) + ((s0 + j) & 31), 64);      // ranges behind the last have none
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += w != 0.f ? w * x[j][e] : 0.f;
        }
    }
    f32x4 o2;
#pragma unroll
    for (int e = 0; e < 4; ++e) o2[e] = __shfl_xor(acc[e], 32, 64);
    float ss = 0.f;
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e] = acc[e] - lam * o2[e];                      // of use in lanes 0..31
        ss += o[e] * o[e];
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) ss += __shfl_xor(ss, x, 64);
    const size_t at = ((size_t)b * a.Nq + i), off = at * a.H * HV + (size_t)h * HV + d;
    if (f.o && m) *(u32x2*)(f.o2 + off) = u32x2{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
    if (f.o && sl == 0) f.lse2[(size_t)m * rows + row] = lse;
    if (m) return;
    if (f.o) *(u32x2*)(f.o + off) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
    if (a.gamma) {
        const float rn = a.out_scale / sqrtf(ss * (1.f / HV) + a.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= rn * gam[e];
    }
    *(u32x2*)(f.out + at * f.ldo + (size_t)h * HV + d) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

// ------------------------------------------------------------------------------------------------ backward
// Row pass: dO from dY through the norm, the four numbers per row that the two big passes need, and the parameters' gradients.
//   g = out_scale * gamma * dY, xhat = O / rms, dO = (g - xhat * mean(g xhat)) / rms;  dgamma += out_scale * dY * xhat
//   d1 = dO . O1, d2 = dO . O2 (O1 = O + lam O2);  dlam -= d2
// stats[b, h, i] = (-lse_1 / c, -(lse_2 - log2|lam|) / c, -d1, d1 - d2), c = scale log2(e): what the score and G accumulators start from, so that
// P1 = exp2(c acc), |lam| P2 = exp2(c acc) and G - d1, G - d2 come out of the matrix instructions.
// 16 lanes a row, a block's rows all of one head; block partials of dgamma / dlam, summed in order by param_block.
// A copy's work: 32 x 1568 x 3 heads 31 us, 5.0 TB/s (one row at a time 35, four, with half the waves, 38).
constexpr int ROWS_AT_ONCE = 2;
__global__ __launch_bounds__(256) void diff_rows_kernel(DiffArgs a, const bf16_t* __restrict__ o, const bf16_t* __restrict__ o2, const bf16_t* __restrict__ dout,
                                                        size_t lddo, const float* __restrict__ lse2, bf16_t* __restrict__ d_o, f32x4* __restrict__ stats,
                                                        float* __restrict__ part, float* __restrict__ lams) {
    __shared__ float red[16][HV + 1];
    const int tid = threadIdx.x, lane = tid & 63, sub = tid & 15, slot = tid >> 4, h = blockIdx.y, nb = gridDim.x;
    float e1, e2;
    const float lam = head_lambda(a, h, lane, e1, e2);
    if (blockIdx.x == 0 && tid == 0) lams[h] = lam;
    const float loglam = fmaxf(fast_log2(fabsf(lam)), -EMPTY_LSE), ic = 1.0f / a.c;    // lam = 0: |lam| P2 = exp2(-1e30) = 0
    float gam[8], dg[8], dl = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        gam[e] = a.gamma ? a.out_scale * param(a.gamma, a.param_bf16, 8 * sub + e) : 1.f;
        dg[e] = 0.f;
    }
    const size_t total = (size_t)a.B * a.Nq, HW = (size_t)a.H * HV, plane = (size_t)a.B * a.H * a.Nq;
    for (size_t base = (size_t)blockIdx.x * (16 * ROWS_AT_ONCE); base < total; base += (size_t)nb * (16 * ROWS_AT_ONCE)) {
        // both rows' loads first; a group behind the last row works on that row and stores nothing
        u32x4 wo[ROWS_AT_ONCE], w2[ROWS_AT_ONCE], wd[ROWS_AT_ONCE];
        float l1[ROWS_AT_ONCE], l2[ROWS_AT_ONCE];
        size_t st[ROWS_AT_ONCE], off[ROWS_AT_ONCE];
        bool some[ROWS_AT_ONCE];
#pragma unroll
        for (int j = 0; j < ROWS_AT_ONCE; ++j) {
            const size_t want = base + 16 * j + slot, row = want < total ? want : total - 1;
            const int b = (int)(row / a.Nq), i = (int)(row - (size_t)b * a.Nq);
            st[j] = ((size_t)b * a.H + h) * a.Nq + i;
            off[j] = row * HW + (size_t)h * HV + 8 * sub;
            wo[j] = *(const u32x4*)(o + off[j]);
            w2[j] = *(const u32x4*)(o2 + off[j]);
            wd[j] = *(const u32x4*)(dout + row * lddo + (size_t)h * HV + 8 * sub);
            l1[j] = lse2[st[j]];
            l2[j] = lse2[plane + st[j]];
            some[j] = row_lim(a, clip_len(a, b), i) > 0;
        }
#pragma unroll
        for (int j = 0; j < ROWS_AT_ONCE; ++j) {
            const bool mine = base + 16 * j + slot < total;
            float vo[8], v2[8], vd[8], gg[8];
            float ss = 0.f, gx = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                vo[e] = (e & 1) ? bf16hi_to_f32(wo[j][e >> 1]) : bf16lo_to_f32(wo[j][e >> 1]);
                v2[e] = (e & 1) ? bf16hi_to_f32(w2[j][e >> 1]) : bf16lo_to_f32(w2[j][e >> 1]);
                vd[e] = (e & 1) ? bf16hi_to_f32(wd[j][e >> 1]) : bf16lo_to_f32(wd[j][e >> 1]);
                gg[e] = gam[e] * vd[e];
                ss += vo[e] * vo[e];
                gx += gg[e] * vo[e];
            }
            u32x4 rd = wd[j];
            if (a.gamma) {
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) {
                    ss += __shfl_xor(ss, x, 64);
                    gx += __shfl_xor(gx, x, 64);
                }
                const float rn = 1.0f / sqrtf(ss * (1.f / HV) + a.eps);
                const float k = gx * rn * rn * (1.f / HV);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (mine && some[j]) dg[e] += a.out_scale * vd[e] * vo[e] * rn;    // not 0 times whatever dout holds there
                    gg[e] = some[j] ? rn * (gg[e] - vo[e] * k) : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) rd[e] = pack_bf16x2(gg[2 * e], gg[2 * e + 1]);
                if (mine) *(u32x4*)(d_o + off[j]) = rd;
            }
            // d1, d2 from the rounded dO that the products read (their rows then sum to zero as the formula's do); dlam from the unrounded
            float d1 = 0.f, d2 = 0.f, dx = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = (e & 1) ? bf16hi_to_f32(rd[e >> 1]) : bf16lo_to_f32(rd[e >> 1]);
                d1 += q * (vo[e] + lam * v2[e]);
                d2 += q * v2[e];
                dx += gg[e] * v2[e];
            }
            if (mine && some[j]) dl -= dx;
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) {
                d1 += __shfl_xor(d1, x, 64);
                d2 += __shfl_xor(d2, x, 64);
            }
            if (sub == 0 && mine) stats[st[j]] = some[j] ? f32x4{-l1[j] * ic, (loglam - l2[j]) * ic, -d1, d1 - d2} : f32x4{-EMPTY_LSE * ic, -EMPTY_LSE * ic, 0.f, 0.f};
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[slot][8 * sub + e] = dg[e];
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) dl += __shfl_xor(dl, x, 64);
    if (sub == 0) red[slot][HV] = dl;
    __syncthreads();
    if (tid <= HV) {
        float t = 0.f;
        for (int k = 0; k < 16; ++k) t += red[k][tid];
        part[((size_t)h * nb + blockIdx.x) * (HV + 1) + tid] = t;
    }
}

// The sums of the parameters' partials, dK / dV and dQ need nothing of each other: one launch, in this order (the longest blocks early, the
// last round of each filled by the next).  32 x 160 x 6 heads 31 us (three launches 16 + 19 + 5), 8 ragged clips of 1111 92 (44 + 70 + 5),
// 32 x 1568 x 3 heads 468 (205 + 270 + 7).
struct GradArgs {
    DiffArgs a;
    const bf16_t* d_o;                                    // dO behind the norm
    size_t lddo;
    const f32x4* stats;
    const float *lams, *part;
    bf16_t *dq, *dk, *dv;
    size_t lddq, lddk, lddv;
    void *dlam, *dgamma;
    int nb, grad_bf16, params, np, nxk, nk, nxq, spread;  // np, nk: the first parts' blocks, multiples of 8 (a block's XCD is its index mod 8)
};
// The kernel's arguments, read where they are used: those of all three parts, and the outputs' through the loops, do not fit the scalar registers
__device__ __forceinline__ const GradArgs& grad_args() {
    auto p = (const __attribute__((address_space(4))) GradArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const GradArgs*)p;
}

// block 0 .. lam_heads - 1: the four vectors' gradients of a head (or of all heads); 16 more blocks: 8 columns of dgamma each.  A block's
// 32 groups of 8 threads walk the partial rows in strides of 32, in a fixed order.
__device__ __forceinline__ void param_block(int id, double* red) {
    const GradArgs& g = grad_args();
    const DiffArgs a = g.a;
    const float* part = g.part;
    const int nb = g.nb, grad_bf16 = g.grad_bf16;
    void *dlam = g.dlam, *dgamma = g.dgamma;
    const int tid = threadIdx.x;
    auto put = [&](void* p, size_t i, float v) {
        if (grad_bf16) ((bf16_t*)p)[i] = f32_to_bf16(v);
        else ((float*)p)[i] = v;
    };
    const bool lam_block = id < a.lam_heads;
    const int first = lam_block && a.lam_heads > 1 ? id : 0, n = (lam_block && a.lam_heads > 1 ? 1 : a.H) * nb;
    const int col = lam_block ? HV : 8 * (id - a.lam_heads) + (tid & 7), start = lam_block ? tid : tid >> 3, step = lam_block ? 256 : 32;
    const float* p = part + (size_t)first * nb * (HV + 1) + col;
    double s = 0.0;
    int k = start;
    for (; k + 7 * step < n; k += 8 * step) {             // eight loads in flight
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[(size_t)(k + e * step) * (HV + 1)];
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)x[e];
    }
    for (; k < n; k += step) s += (double)p[(size_t)k * (HV + 1)];
    red[tid] = s;
    __syncthreads();
    for (int o = 128; o >= (lam_block ? 1 : 8); o >>= 1) {
        if (tid < o) red[tid] += red[tid + o];
        __syncthreads();
    }
    if (lam_block) {
        const float dl = (float)red[0];
        float e1, e2;
        head_lambda(a, id, tid & 63, e1, e2);
        const int v = tid >> 6;                                    // wave v: vector v; its partner is v ^ 1
        const size_t st = (size_t)a.lam_heads * 64, at = (size_t)id * 64 + (tid & 63);
        put(dlam, v * st + at, dl * (v < 2 ? e1 : -e2) * param(a.lam, a.param_bf16, (v ^ 1) * st + at));
    } else if (tid < 8) {
        put(dgamma, col, (float)red[tid]);
    }
}

// dQ: dS_m = P_m (G - d_m), G = dO V^T; dQ_1 = scale dS_1 K_1, dQ_2 = -lam scale dS_2 K_2 (|lam| sits in the probability)
// Blocks and rings as in the forward pass; 24 matrix instructions and 24 KiB of LDS reads a tile and wave.  Alone 32 x 1568 x 3 heads 205 us,
// 590 TFLOP/s.
constexpr int dq_lds(bool keys4) { return 16 * TILE + (keys4 ? OUT_WAVE : 0); }
template <bool KEYS4>
__device__ __forceinline__ void dq_block(int id, unsigned char* smem) {
    const GradArgs& in = grad_args();
    const DiffArgs a = in.a;
    const bf16_t* __restrict__ d_o = in.d_o;
    const size_t lddo = in.lddo;
    const f32x4* __restrict__ stats = in.stats;
    const float* __restrict__ lams = in.lams;
    constexpr int STAGE = 4 * TILE, ROWS = KEYS4 ? 32 : 128;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int xb, b, kvh;
    if (!place_block(a, id, in.nxq, in.spread, true, xb, b, kvh)) return;
    const int len = clip_len(a, b);
    const int rb0 = a.row0 + xb * ROWS, r0 = rb0 + (KEYS4 ? 0 : wave * 32);
    const Row w = make_row(a, kvh, r0 + (lane & 31), len);
    int wlo = 0, whi = 0, blo, bhi;
    span_lim(a, len, rb0, min(rb0 + ROWS, a.R) - 1, blo, bhi);
    if (r0 < a.R) span_lim(a, len, r0, min(r0 + 32, a.R) - 1, wlo, whi);
    const int all = (bhi + 31) >> 5, first = KEYS4 ? wave : 0, stride = KEYS4 ? 4 : 1, nkt = KEYS4 ? (all - wave + 3) >> 2 : all;
    const size_t kr = (size_t)b * a.Nk;
    const bf16_t *kp = a.k + kr * a.ldk + (size_t)kvh * HV, *vp = a.v + kr * a.ldv + (size_t)kvh * HV;
    HalfTile ht = half_tile((KEYS4 || wave < 2 ? kp : vp) + (KEYS4 ? 0 : (wave & 1) * 64), KEYS4 || wave < 2 ? a.ldk : a.ldv, lane), hv;
    if constexpr (KEYS4) hv = half_tile(vp, a.ldv, lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem), ring = KEYS4 ? wave * STAGE : 0;
    auto issue = [&](int t, unsigned buf) {
        const int row0 = (first + t * stride) * 32;
        const unsigned at = lds0 + ring + buf * STAGE;
        if constexpr (KEYS4) {
            dma_tiles(ht, hv, row0, len, at, lane);
        } else {
            dma_half_tile(ht, row0, len, at + wave * TILE, lane);
        }
    };
    if (nkt > 0) issue(0, 0);
    if (!KEYS4 && nkt > 1) issue(1, 1);
    bf16x8 qf[2][4], of[8];
    const bf16_t* qp = a.q + row_at(a, b, w) * a.ldq + (size_t)w.h * HV;
    const bf16_t* op = d_o + row_at(a, b, w) * lddo + (size_t)w.h * HV;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[m][ks] = *(const bf16x8*)(qp + 64 * m + 16 * ks + 8 * hh);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) of[ks] = *(const bf16x8*)(op + 16 * ks + 8 * hh);
    const f32x4 rs = stats[stat_at(a, b, w)];
    const float nl[2] = {rs[0] * a.c, rs[1] * a.c}, nd[2] = {rs[2], rs[2] + rs[3]};
    f32x16 dqa[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m) dqa[m][0] = dqa[m][1] = zero16();
    const FragOff fo = frag_off(lds0 + ring, lane);
    for (int t = 0; t < nkt; ++t) {
        if constexpr (KEYS4) {
            landed_own();
        } else if ((t & 1) == 0) {
            landed_barrier<0>();
            if (t + 2 < nkt) issue(t + 2, (t + 2) & 3);
            if (t + 3 < nkt) issue(t + 3, (t + 3) & 3);
        }
        const int k0 = (first + t * stride) * 32;
        const unsigned T = (KEYS4 ? 0 : t & 3) * STAGE;
        if (k0 >= whi) continue;
        bf16x8 fr[4];
        RowOff ro(fo, T);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) fr[ks] = ro.get(0, ks);
        f32x16 s[2] = {zero16(), zero16()}, g = zero16();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            s[0] = mfma(fr[ks], qf[0][ks], s[0]);
            fr[ks] = ro.get(2 * TILE, ks);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            g = mfma(fr[ks], of[ks], g);
            fr[ks] = ro.get(3 * TILE, ks);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            g = mfma(fr[ks], of[4 + ks], g);
            fr[ks] = ro.get(TILE, ks);
        }
        ColOff co(fo, T);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            s[1] = mfma(fr[ks], qf[1][ks], s[1]);
            fr[ks] = co.get(0, ks >> 1, ks & 1);
        }
        if (k0 + 32 > wlo) {
            int lim = w.lim - k0 - 4 * hh;
            asm volatile("" : "+v"(lim));
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((r & 3) + 8 * (r >> 2) >= lim) s[0][r] = s[1][r] = -__builtin_inff();
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (KEYS4 && m == 1) {
                reads_done();
                if (t + 1 < nkt) issue(t + 1, 0);
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                float p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) p[r] = fast_exp2(fmaf(s[m][8 * s2 + r], a.c, nl[m])) * (g[8 * s2 + r] + nd[m]);
                const bf16x8 f = pack_frag(p, 0);
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) {
                    dqa[m][dt] = mfma(fr[2 * s2 + dt], f, dqa[m][dt]);
                    if (m == 0) fr[2 * s2 + dt] = co.get(TILE, s2, dt);
                }
            }
        }
    }
    const bool some = w.lim > 0;
    const float m1 = some ? a.scale : 0.f, m2 = lams[w.h] < 0.f ? m1 : -m1;
    if (!some) {                                          // not times zero: a row that sees nothing may hold NaN
#pragma unroll
        for (int m = 0; m < 2; ++m) dqa[m][0] = dqa[m][1] = zero16();
    }
    __syncthreads();                                      // the ring is free
    const GradArgs& fin = grad_args();
    bf16_t* dq = fin.dq;
    const size_t lddq = fin.lddq;
    if constexpr (KEYS4) {
        unsigned char* mine = smem + wave * STAGE;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            acc_put(mine, dt, lane, dqa[0][dt], m1);
            acc_put(mine, 2 + dt, lane, dqa[1][dt], m2);
        }
        __syncthreads();
        out_put16(smem + 4 * STAGE, lane, wave, acc_sum(smem, STAGE, wave, lane), 1.f);
        __syncthreads();
        out_flush(smem + 4 * STAGE, lane, [&](int r) { return list_row(a, dq, lddq, b, kvh, r0 + r); }, 2 * wave, 2 * wave + 2);
    } else {
        unsigned char* lds = smem + wave * OUT_WAVE;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            out_put16(lds, lane, dt, dqa[0][dt], m1);
            out_put16(lds, lane, 2 + dt, dqa[1][dt], m2);
        }
        out_flush(lds, lane, [&](int r) { return list_row(a, dq, lddq, b, kvh, r0 + r); });
    }
}

// dK, dV: a wave owns 32 keys and walks the query rows of its key head's G heads.  dV = A^T dO with A = P1 - lam P2,
// dK_1 = scale dS_1^T Q_1, dK_2 = -lam scale dS_2^T Q_2.  Rows that see nothing are staged as zeros, with a log-sum of 1e30.
// 128 accumulator registers leave no room for two waves a SIMD with both K and V in registers: V stays in LDS (32 KiB a block), and the
// dV product comes before G = dO V^T, so that A is gone when G needs its place.  Two LDS stages of Q, dO and the rows' statistics.
// A row's statistics are wanted by every lane of an accumulator row: each lane splits its own row's numbers into three bf16 terms (exact to
// f32) and one more matrix instruction, against a selector of ones, spreads a number over the accumulator.  Reading them from LDS per
// accumulator row cost as much LDS time as two operands.  Alone 32 x 1568 x 3 heads 270 us: matrix unit 45 % and vector unit 44 % busy.
__device__ const f32x4 g_pad_stat = {-1.0e36f, -1.0e36f, 0.f, 0.f};     // a row behind the last: exp2(c acc) = 0
__device__ __forceinline__ bf16x8 split3(float x, float y) {
    u32x4 f = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 3; ++e) {
        const uint32_t w = pack_bf16x2(x, y);
        f[e] = w;
        x -= bf16lo_to_f32(w);
        y -= bf16hi_to_f32(w);
    }
    return __builtin_bit_cast(bf16x8, f);
}
__device__ __forceinline__ bf16x8 selector(uint32_t w) {
    asm volatile("" : "+v"(w));                                           // made anew where it is used: four hoisted ones are 16 registers
    return __builtin_bit_cast(bf16x8, u32x4{w, w, w, w});
}

constexpr int DKV_BUF = 4 * TILE + 512;
constexpr int dkv_lds(bool rows4) { return rows4 ? 4 * DKV_BUF + 2 * TILE + 1024 : 2 * DKV_BUF + 8 * TILE; }
template <bool ROWS4>
__device__ __forceinline__ void dkv_block(int id, unsigned char* smem) {
    const GradArgs& in = grad_args();
    const DiffArgs a = in.a;
    const bf16_t* __restrict__ d_o = in.d_o;
    const size_t lddo = in.lddo;
    const f32x4* __restrict__ stats = in.stats;
    const float* __restrict__ lams = in.lams;
    constexpr int BUF = DKV_BUF, VAT = (ROWS4 ? 4 : 2) * BUF;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int xb, b, kvh;
    if (!place_block(a, id, in.nxk, in.spread, false, xb, b, kvh)) return;
    const int len = clip_len(a, b), off = past(a, len);
    const int kb0 = xb * (ROWS4 ? 32 : 128), k0 = kb0 + (ROWS4 ? 0 : wave * 32), key = k0 + (lane & 31);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem);
    const unsigned ring = ROWS4 ? wave * BUF : 0, vt = VAT + (ROWS4 ? 0 : wave * 2 * TILE);
    const FragOff fo = frag_off(lds0, lane);
    {
        const bf16_t* vp = a.v + (size_t)b * a.Nk * a.ldv + (size_t)kvh * HV;
        if (!ROWS4 || wave == 0) {
            dma_half_tile(half_tile(vp, a.ldv, lane), k0, len, lds0 + vt, lane);
            dma_half_tile(half_tile(vp + 64, a.ldv, lane), k0, len, lds0 + vt + TILE, lane);
        }
    }
    bf16x8 kf[2][4];
    const bf16_t* kp = a.k + ((size_t)b * a.Nk + (key < a.Nk ? key : a.Nk - 1)) * a.ldk + (size_t)kvh * HV;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
        u32x4 x = *(const u32x4*)(kp + 16 * ks + 8 * hh);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = key < len ? x[e] : 0u;         // whatever a row behind the clip's last one holds
        kf[ks >> 2][ks & 3] = __builtin_bit_cast(bf16x8, x);
    }
    f32x16 dva[4], dka[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        dva[i] = zero16();
        dka[i >> 1][i & 1] = zero16();
    }
    const int nqt = (a.Nq + 31) >> 5;
    // the query tiles in which some row sees the block's first key: limits grow with i
    const int q_first = kb0 >= len ? nqt : min(max(kb0 - off + 1, 0) >> 5, nqt);
    const int row_first = min(max(1 - off, 0), a.Nq);                     // rows in front of it see nothing
    const int per = nqt - q_first, all = per * a.G, stride = ROWS4 ? 4 : 1, steps = ROWS4 ? (all - wave + 3) >> 2 : all;
    const bf16_t *qbase = a.q + (size_t)b * a.Nq * a.ldq, *obase = d_o + (size_t)b * a.Nq * lddo;
    HalfTile ht = half_tile(ROWS4 || wave < 2 ? qbase : obase, ROWS4 || wave < 2 ? a.ldq : lddo, lane), ho;
    if constexpr (ROWS4) ho = half_tile(obase, lddo, lane);
    auto issue = [&](int g, int qt, unsigned buf) {
        const int h = kvh * a.G + g;
        const unsigned at = lds0 + ring + buf * BUF;
        HalfTile hi = ht;
        hi.base += (size_t)h * HV;
        if constexpr (ROWS4) {
            HalfTile yi = ho;
            yi.base += (size_t)h * HV;
            dma_tiles(hi, yi, qt * 32, a.Nq, at, lane, row_first);
        } else {
            hi.base += (wave & 1) * 64;
            dma_half_tile(hi, qt * 32, a.Nq, at + wave * TILE, lane, row_first);
        }
        int row = lane;
        asm volatile("" : "+v"(row));
        if ((ROWS4 || wave == 0) && row < 32) {
            const int i = qt * 32 + row;
            dma_b128(i < a.Nq ? (const void*)(stats + ((size_t)b * a.H + h) * a.Nq + i) : (const void*)&g_pad_stat, at + 4 * TILE);
        }
    };
    // this step's head and tile, the next one's: all tiles of a head, then the next head's; ROWS4 in strides of four
    int g = 0, qt = q_first, ng = 0, nqt_next = q_first;
    auto advance = [&](int& gg, int& tt, int by) {
        tt += by;
        while (tt >= nqt && gg < a.G) {
            tt -= per;
            ++gg;
        }
    };
    if (ROWS4 && per > 0) {
        advance(g, qt, wave);
        ng = g;
        nqt_next = qt;
    }
    float sgn = 1.f;
    int sgn_of = -1;
    if (steps > 0) {
        issue(g, qt, 0);
        advance(ng, nqt_next, stride);
    }
    if (ROWS4) landed_barrier<0>();                                       // V is everybody's
    else if (steps == 0) landed_barrier<0>();                             // V's pieces must not outlive the block
    // selectors: the lower half of the lanes offers the score terms, the upper half those of G
    const uint32_t lower = hh ? 0u : ~0u;
    auto step = [&](int t, auto buf_tag) {
        constexpr int PAR = decltype(buf_tag)::value;
        if constexpr (ROWS4) landed_own();
        else landed_barrier<0>();
        if (!ROWS4 && t + 1 < steps) issue(ng, nqt_next, 1 - PAR);
        if (g != sgn_of) {                                                // a head begins
            sgn = lams[kvh * a.G + g] < 0.f ? -1.f : 1.f;
            sgn_of = g;
        }
        const unsigned T = ring + PAR * BUF;
        const int i0 = qt * 32, last = min(i0 + 31, a.Nq - 1);
        const int gi = ng, qi = nqt_next;
        advance(g, qt, stride);
        advance(ng, nqt_next, stride);
        auto refill = [&]() {
            if (ROWS4) {
                reads_done();
                if (t + 1 < steps) issue(gi, qi, 0);
            }
        };
        if (min(len, last + off) <= k0) {
            refill();
        } else {
            // four fragment registers: each is refilled right behind the matrix instruction that read it, a group ahead
            bf16x8 fr[4];
            RowOff ro(fo);
            const f32x4 rs = *(const LDS_AS f32x4*)(size_t)(lds0 + T + 4 * TILE + (lane & 31) * 16);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) fr[ks] = ro.get(T, ks);
            const bf16x8 st = split3(hh ? rs[2] : rs[0], hh ? rs[3] : rs[1]);
            f32x16 s1 = mfma(st, selector(lower & 0x00003f80u), zero16()), s2 = mfma(st, selector(lower & 0x3f800000u), zero16());
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                s1 = mfma(fr[ks], kf[0][ks], s1);
                fr[ks] = ro.get(T + TILE, ks);
            }
            ColOff co(fo);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                s2 = mfma(fr[ks], kf[1][ks], s2);
                fr[ks] = co.get(T + (2 + (ks >> 1)) * TILE, 0, ks & 1);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s1[r] = fast_exp2(s1[r] * a.c);
#pragma unroll
            for (int r = 0; r < 16; ++r) s2[r] = fast_exp2(s2[r] * a.c);
            if (min(len, i0 + off) < k0 + 32) {                           // hidden: key >= len or i <= key - off
                int t = key >= len ? 1 << 30 : key - off - i0 - 4 * hh;
                asm volatile("" : "+v"(t));
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if ((r & 3) + 8 * (r >> 2) <= t) s1[r] = s2[r] = 0.f;
            }
            {
                float A[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) A[r] = fmaf(-sgn, s2[r], s1[r]);
                const bf16x8 fa0 = pack_frag(A, 0), fa1 = pack_frag(A, 1);
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    dva[dt] = mfma(fr[dt], fa0, dva[dt]);
                    fr[dt] = co.get(T + (2 + (dt >> 1)) * TILE, 1, dt & 1);
                    
                }
                ro = RowOff(fo);
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    dva[dt] = mfma(fr[dt], fa1, dva[dt]);
                    fr[dt] = (dt & 1) ? ro.get(vt, dt >> 1) : ro.get(T + 2 * TILE, dt >> 1);
                    
                }
            }
            co = ColOff(fo);
            f32x16 gr = mfma(st, selector(~lower & 0x00003f80u), zero16());
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const int x = 2 * (ks & 1), n = ks + 2;
                gr = mfma(fr[x], fr[x + 1], gr);
                if (n < 8) {
                    fr[x] = ro.get(T + (2 + (n >> 2)) * TILE, n & 3);
                    fr[x + 1] = ro.get(vt + (n >> 2) * TILE, n & 3);
                } else {
                    fr[x] = co.get(T, ks & 1, 0);
                    fr[x + 1] = co.get(T, ks & 1, 1);
                }
            }
            {
                float p1[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) p1[r] = s1[r] * gr[r];
                const bf16x8 f0 = pack_frag(p1, 0), f1 = pack_frag(p1, 1);
                gr = mfma(st, selector(~lower & 0x3f800000u), gr);        // G - d1 -> G - d2
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int dt = 0; dt < 2; ++dt) {
                        dka[0][dt] = mfma(fr[2 * s + dt], s ? f1 : f0, dka[0][dt]);
                        fr[2 * s + dt] = co.get(T + TILE, s, dt);
                        
                    }
            }
            refill();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float p2[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) p2[r] = s2[8 * s + r] * gr[8 * s + r];
                u32x4 f2 = __builtin_bit_cast(u32x4, pack_frag(p2, 0));
                if (sgn < 0.f) f2 ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
                dka[1][0] = mfma(fr[2 * s], __builtin_bit_cast(bf16x8, f2), dka[1][0]);
                dka[1][1] = mfma(fr[2 * s + 1], __builtin_bit_cast(bf16x8, f2), dka[1][1]);
            }
        }
    };
    for (int t = 0; t < steps; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < steps) step(t + 1, std::integral_constant<int, ROWS4 ? 0 : 1>{});
    }
    __syncthreads();                                      // the stages are free
    int l = lane;
    asm volatile("" : "+v"(l));                           // nothing of this is kept through the loop
    const GradArgs& fin = grad_args();
    bf16_t *dk = fin.dk, *dv = fin.dv;
    const size_t lddk = fin.lddk, lddv = fin.lddv, row0 = (size_t)b * fin.a.Nk;
    const int Nk = fin.a.Nk;
    const float scale = fin.a.scale;
    auto dk_row = [&](int r) { return k0 + r < Nk ? dk + (row0 + k0 + r) * lddk + (size_t)kvh * HV : (bf16_t*)nullptr; };
    auto dv_row = [&](int r) { return k0 + r < Nk ? dv + (row0 + k0 + r) * lddv + (size_t)kvh * HV : (bf16_t*)nullptr; };
    if constexpr (ROWS4) {
        // dK, then dV: there is no room for both
        unsigned char *mine = smem + wave * 4 * 4096, *out = smem + VAT;
        static_assert(OUT_WAVE <= 2 * TILE + 1024 && 4 * 4 * 4096 <= VAT, "the sums and the rows that leave have their places");
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) acc_put(mine, dt, l, pass ? dva[dt] : dka[dt >> 1][dt & 1], pass ? 1.f : dt < 2 ? scale : -scale);
            __syncthreads();
            out_put16(out, l, wave, acc_sum(smem, 4 * 4096, wave, l), 1.f);
            __syncthreads();
            if (pass) out_flush(out, l, dv_row, 2 * wave, 2 * wave + 2);
            else out_flush(out, l, dk_row, 2 * wave, 2 * wave + 2);
            __syncthreads();
        }
    } else {
        unsigned char* lds = smem + wave * OUT_WAVE;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            out_put16(lds, l, dt, dka[0][dt], scale);
            out_put16(lds, l, 2 + dt, dka[1][dt], -scale);
        }
        out_flush(lds, l, dk_row);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) out_put16(lds, l, dt, dva[dt], 1.f);
        out_flush(lds, l, dv_row);
    }
}

template <bool KEYS4, bool ROWS4>
__global__ __launch_bounds__(256, 2) void diff_grad_kernel(GradArgs) {
    constexpr int LDS_Q = dq_lds(KEYS4), LDS_K = dkv_lds(ROWS4);
    __shared__ __attribute__((aligned(128))) unsigned char smem[LDS_Q > LDS_K ? LDS_Q : LDS_K];
    const GradArgs& g = grad_args();
    const int id = blockIdx.x, np = g.np, nk = g.nk;
    if (id < np) {
        if (id < g.params) param_block(id, (double*)smem);
    } else if (id < np + nk) {
        dkv_block<ROWS4>(id - np, smem);
    } else {
        dq_block<KEYS4>(id - np - nk, smem);
    }
}

// ------------------------------------------------------------------------------------------------ host
int check(const char* who, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int B, int Nq, int Nk, int H, int Hkv, float scale,
          const void* lam, int lam_heads, int causal, bool norm, float eps) {
    if (!q || !k || !v || !lam) MOFO_FAIL(MOFO_EINVAL, "%s: null pointer", who);
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv)
        MOFO_FAIL(MOFO_EINVAL, "%s: bad dims B=%d Nq=%d Nk=%d H=%d Hkv=%d (H a multiple of Hkv)", who, B, Nq, Nk, H, Hkv);
    if (H > 4096) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: H=%d (at most 4096)", who, H);
    // beyond them EMPTY_LSE over the exponent's factor, or a score times it, leaves f32
    if (!(scale >= 0x1p-24f && scale <= 0x1p24f)) MOFO_FAIL(MOFO_EINVAL, "%s: scale must lie in 2^-24 .. 2^24", who);
    if (norm && !(eps >= 0x1p-100f && eps < 3.0e38f)) MOFO_FAIL(MOFO_EINVAL, "%s: eps must be at least 2^-100 (a row of zeros has no root mean square)", who);
    if (lam_heads != 1 && lam_heads != H) MOFO_FAIL(MOFO_EINVAL, "%s: lam of %d heads, must be 1 or H=%d", who, lam_heads, H);
    if (causal < 0 || causal > 2) MOFO_FAIL(MOFO_EINVAL, "%s: causal=%d must be 0, 1 or 2", who, causal);
    if (ldq < H * HV || ldk < Hkv * HV || ldv < Hkv * HV || (ldq | ldk | ldv) % 8)
        MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: bad leading dims ldq=%d ldk=%d ldv=%d (multiples of 8, a row of 128 columns a head)", who, ldq, ldk, ldv);
    if (ldk > (1 << 24) || ldv > (1 << 24) || ldq > (1 << 24)) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: row pitch above 2^24", who);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: q, k, v must be 16-byte aligned", who);
    if ((long long)(H / Hkv) * Nq > (1LL << 30) || Nk > (1 << 30)) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: too many rows", who);
    if ((long long)B * Hkv * (((long long)(H / Hkv) * Nq + Nk) / 32 + 2) > (1LL << 28)) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: grid too large", who);
    return MOFO_OK;
}
int check_blocks(const char* who, long long blocks) {
    if (blocks > MOFO_MAX_BLOCKS_256) MOFO_FAIL(MOFO_EUNSUPPORTED, "%s: %lld blocks of a launch (at most %lld)", who, blocks, MOFO_MAX_BLOCKS_256);
    return MOFO_OK;
}

DiffArgs make_args(const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int B, int Nq, int Nk, int H, int Hkv, float scale,
                   const void* lam, int lam_heads, float lam_init, const void* gamma, int param_bf16, float eps, float out_scale, const int* kv_len, int causal) {
    DiffArgs a;
    a.q = (const bf16_t*)q;
    a.k = (const bf16_t*)k;
    a.v = (const bf16_t*)v;
    a.ldq = (size_t)ldq;
    a.ldk = (size_t)ldk;
    a.ldv = (size_t)ldv;
    a.B = B;
    a.H = H;
    a.Hkv = Hkv;
    a.G = H / Hkv;
    a.Nq = Nq;
    a.Nk = Nk;
    a.R = a.G * Nq;
    a.causal = causal;
    a.row0 = 0;
    a.kv_len = kv_len;
    a.lam = lam;
    a.gamma = gamma;
    a.param_bf16 = param_bf16;
    a.lam_heads = lam_heads;
    a.lam_init = lam_init;
    a.scale = scale;
    a.c = scale * 1.4426950408889634f;
    a.eps = eps;
    a.out_scale = out_scale;
    return a;
}

constexpr int PART = 2 * HV + 4;        // floats of workspace per row and range

// Which block form, from a model of the time on 256 compute units that its measurements gave, us:
//   128 rows (keys) a block, `steps` 32 x 32 tiles in a row    6.8 + 0.92 steps, two blocks on a compute unit 1.45 times that
//   KEYS4 / ROWS4, 32 rows, a quarter of the steps             7.6 + 1.28 steps, two 9.9 + 1.7 steps
// two blocks a compute unit at a time, rounds of 512 of them.  Causal blocks of a round differ in length and even out.
// Measured, 128-row against four-way blocks, forward: 6 heads x 1568 52 / 31, 12 heads 53 / 52, 18 heads 54 / 62, 24 heads 74 / 80;
// 32 x 6 heads x 160 17 / 24, 8 x 6 x 320 17 / 16, 4 heads x 16 clips of 50 8.9 / 11; causal 3 heads x 5014 155 / 63, 12 x 2500 82 / 65.
// dQ follows the forward to a tenth.  dK / dV: 6 heads x 1568 60 / 31; causal 8 x 1111, 4 heads a key head 180 / 70.  A four-way ring of two
// tiles, one block a compute unit, was 1.6 times slower beyond 256 blocks and at most 5 % faster below.
double block_time(bool four, long long blocks, long long tiles, bool causal) {
    const double steps = four ? (double)((tiles + 3) / 4) * (causal ? 0.75 : 1.0) : (double)tiles;
    const double one = four ? 7.6 + 1.28 * steps : 6.8 + 0.92 * steps, two = four ? 9.9 + 1.7 * steps : (causal ? 1.2 : 1.45) * one;
    if (blocks <= 256) return one;
    if (causal) return two * (blocks <= 512 ? 1.0 : blocks / 512.0);
    const long long rest = blocks % 512;
    return (double)(blocks / 512) * two + (rest == 0 ? 0.0 : rest <= 256 ? one : two);
}
bool four_way(long long groups, long long rows, long long tiles, bool causal) {
    return block_time(true, groups * ((rows + 31) / 32), tiles, causal) < block_time(false, groups * ((rows + 127) / 128), tiles, causal);
}
// Equal blocks, `others` of another part in front of them: beyond 512 the rows of the last, partial round may be left to four-way blocks in
// a launch behind the first.  nx 128-row blocks a list.  us, all rows in 128-row blocks, in four-way ones, and 85 blocks and 52 four-way ones
// a list: forward 6 heads x 12544 890 / 848 / 746.
struct Cut {
    long long nx;
    double time;
};
Cut cut_rows(long long others, long long groups, long long rows, long long tiles) {
    const long long n = (rows + 127) / 128, full = (others + groups * n) / 512 * 512 - others, nx = full > 0 ? full / groups : 0;
    const double whole = block_time(false, others + groups * n, tiles, false);
    if (nx <= 0 || nx >= n) return {n, whole};
    const double cut = block_time(false, others + groups * nx, tiles, false) + block_time(true, groups * ((rows - nx * 128 + 31) / 32), tiles, false) + 3.0;
    return cut < whole ? Cut{nx, cut} : Cut{n, whole};
}
int tail_blocks(const Cut& c, long long rows) { return c.nx * 128 < rows ? (int)((rows - c.nx * 128 + 31) / 32) : 0; }

// Forward: four-way blocks may cut the keys into ranges as well (few rows against a long cache), joined by a kernel of its own: 3 us more and a
// little per range, and a partial row is written and read at about 1500 rows a us.  At most 64 ranges and 65536 partial rows.  us by
// ranges: one token against 16 caches of 8192 1 96, 4 36, 8 32, 16 32, 32 36; against one 1 91, 8 21, 32 16, 64 18; 11 rows x 1700 keys x
// 36 heads 1 27, 6 17, 16 23; one head x 1568 1 24, 4 20, 8 22.
struct FwdPlan {
    bool keys4;
    int nx, nsplit, tail;     // tail: four-way blocks a list behind nx * 128 rows, in a launch of their own
};
FwdPlan fwd_plan(int B, int Nq, int Nk, int H, int Hkv, int causal) {
    const long long R = (long long)(H / Hkv) * Nq, rows = (long long)B * H * Nq, groups = (long long)B * Hkv, tiles = (Nk + 31) / 32;
    const long long n1 = (R + 127) / 128, n4 = (R + 31) / 32;
    const bool half = causal == 1;                        // towards the end: every row sees nearly all keys
    const Cut c = half ? Cut{n1, block_time(false, groups * n1, tiles, true)} : cut_rows(0, groups, R, tiles);
    FwdPlan p = {false, (int)c.nx, 1, tail_blocks(c, R)};
    double best = c.time;
    for (int n = 1; n <= 64 && (n == 1 || (n <= tiles && n * rows <= 65536)); ++n) {
        const double t = block_time(true, groups * n4 * n, (tiles + n - 1) / n, half) + (n > 1 ? 3.0 + 0.05 * n + n * rows / 1500.0 : 0.0);
        if (t < best) {
            best = t;
            p = {true, (int)n4, n, 0};
        }
    }
    return p;
}
// place_block: over all XCDs when lengths differ, or with few causal heads; eighths of the list otherwise, where K / V stay in one L2.  us,
// eighths against spread, forward / gradient: 16 x 6 heads x 1568 241 / 501 against 248 / 506; one clip of 12544 925 / 2063, 940 / 2158;
// causal 6 heads x 5014 111 / 214, 96 / 214, 8 heads 120 / 257, 122 / 259, 12 heads 169 / 369, 170 / 336; ragged causal 1111, 4 heads a key
// head, 8 clips 60 / 136, 57 / 114, 32 clips 197 / 383, 178 / 364
int spread_of(const DiffArgs& a) {
    return a.kv_len || (a.causal && (long long)a.B * a.Hkv < 16);
}
long long grid_of(const DiffArgs& a, int nx) {
    const long long n = (long long)a.B * a.Hkv * nx;
    return 8 * ((n + 7) / 8);
}
// blocks of one head's rows in the row pass: about 1024 in all, 64 rows each at least
int row_blocks(int B, int Nq, int H) {
    const long long rows = (long long)B * Nq;
    long long nb = (rows + 63) / 64, most = 1024 / H;
    if (most < 1) most = 1;
    return (int)(nb < most ? nb : most);
}

}  // namespace

extern "C" int mofo_diff_attention_fwd(const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int B, int Nq, int Nk, int H, int Hkv,
                                       float scale, const void* lam, int lam_heads, float lam_init, const void* gamma, int param_is_bf16, float eps,
                                       float out_scale, const int* kv_len, int causal, void* out, int ldo, void* o, void* o2, float* lse2,
                                       float* ws, long long ws_elems, void* stream) {
    int rc = check("mofo_diff_attention_fwd", q, ldq, k, ldk, v, ldv, B, Nq, Nk, H, Hkv, scale, lam, lam_heads, causal, gamma != nullptr, eps);
    if (rc) return rc;
    if (!out) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_fwd: null output");
    if (!o != !o2 || !o != !lse2) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_fwd: o, o2 and lse2 go together");
    if (ldo < H * HV || ldo % 8 || (((uintptr_t)out | (uintptr_t)o | (uintptr_t)o2) & 15))
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_diff_attention_fwd: bad ldo=%d (a multiple of 8), or an output that is not 16-byte aligned", ldo);
    const FwdPlan pl = fwd_plan(B, Nq, Nk, H, Hkv, causal);
    const long long rows = (long long)B * H * Nq;
    if (pl.nsplit > 1 && (!ws || ws_elems < rows * pl.nsplit * PART)) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_fwd: ws of %lld floats is too small", ws ? ws_elems : 0);
    if (pl.nsplit > 1 && ((uintptr_t)ws & 15)) MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_diff_attention_fwd: ws must be 16-byte aligned");
    {
        const long long HW = (long long)H * HV * 2, KW = (long long)Hkv * HV * 2, Mq = (long long)B * Nq, Mk = (long long)B * Nk, es = param_is_bf16 ? 2 : 4;
        const MofoSpan outs[] = {{"out", out, Mq, HW, 2LL * ldo}, {"o", o, 1, Mq * HW, 0}, {"o2", o2, 1, Mq * HW, 0}, {"lse2", lse2, 1, 8 * Mq * H, 0},
                                 {"ws", pl.nsplit > 1 ? ws : nullptr, 1, rows * pl.nsplit * PART * 4, 0}};
        const MofoSpan in[] = {{"q", q, Mq, HW, 2LL * ldq}, {"k", k, Mk, KW, 2LL * ldk}, {"v", v, Mk, KW, 2LL * ldv}, {"lam", lam, 1, 256LL * lam_heads * es, 0},
                               {"gamma", gamma, 1, HV * es, 0}, {"kv_len", kv_len, 1, 4LL * B, 0}};
        MOFO_CHECK_APART("mofo_diff_attention_fwd", outs, 5, in, 6);
    }
    DiffArgs a = make_args(q, ldq, k, ldk, v, ldv, B, Nq, Nk, H, Hkv, scale, lam, lam_heads, lam_init, gamma, param_is_bf16, eps, out_scale, kv_len, causal);
    FwdOut f = {(bf16_t*)out, (bf16_t*)o, (bf16_t*)o2, (size_t)ldo, lse2, nullptr, nullptr};
    if (pl.nsplit > 1) {
        f.part = ws;
        f.part_stat = (f32x2*)(ws + rows * pl.nsplit * (2 * HV));
    }
    const int spread = spread_of(a);
    rc = check_blocks("mofo_diff_attention_fwd", std::max(grid_of(a, pl.nx * pl.nsplit), grid_of(a, pl.tail)));
    if (rc) return rc;
    const dim3 grid((unsigned)grid_of(a, pl.nx * pl.nsplit));
    hipStream_t s = (hipStream_t)stream;
    auto four_way_rows = [&](int nx) {
        const dim3 g((unsigned)grid_of(a, nx));
        if (o) hipLaunchKernelGGL((diff_fwd_kernel<true, true, false>), g, dim3(256), 0, s, a, f, nx, 1, spread);
        else hipLaunchKernelGGL((diff_fwd_kernel<true, false, false>), g, dim3(256), 0, s, a, f, nx, 1, spread);
    };
    if (pl.nsplit > 1) {
        if (o) hipLaunchKernelGGL((diff_fwd_kernel<true, true, true>), grid, dim3(256), 0, s, a, f, pl.nx, pl.nsplit, spread);
        else hipLaunchKernelGGL((diff_fwd_kernel<true, false, true>), grid, dim3(256), 0, s, a, f, pl.nx, pl.nsplit, spread);
    } else if (pl.keys4) {
        four_way_rows(pl.nx);
    } else {
        if (o) hipLaunchKernelGGL((diff_fwd_kernel<false, true, false>), grid, dim3(256), 0, s, a, f, pl.nx, 1, spread);
        else hipLaunchKernelGGL((diff_fwd_kernel<false, false, false>), grid, dim3(256), 0, s, a, f, pl.nx, 1, spread);
    }
    if (pl.tail) {
        MOFO_CHECK_LAUNCH("mofo_diff_attention_fwd");
        a.row0 = pl.nx * 128;
        four_way_rows(pl.tail);
    }
    MOFO_CHECK_LAUNCH("mofo_diff_attention_fwd");
    if (pl.nsplit > 1) {
        hipLaunchKernelGGL(diff_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, f, pl.nsplit);
        MOFO_CHECK_LAUNCH("mofo_diff_attention_fwd(join)");
    }
    return MOFO_OK;
}

extern "C" long long mofo_diff_attention_fwd_ws(int B, int Nq, int Nk, int H, int Hkv) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_fwd_ws: bad dims");
    const int n0 = fwd_plan(B, Nq, Nk, H, Hkv, 0).nsplit, n1 = fwd_plan(B, Nq, Nk, H, Hkv, 1).nsplit, n = n0 > n1 ? n0 : n1;
    return n > 1 ? (long long)B * H * Nq * n * PART : 0;
}

extern "C" long long mofo_diff_attention_bwd_ws(int B, int Nq, int Nk, int H, int Hkv, int norm) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_bwd_ws: bad dims");
    const long long rows = (long long)B * Nq * H;
    return rows * 4 + (norm ? rows * (HV / 2) : 0) + (long long)H * row_blocks(B, Nq, H) * (HV + 1) + H;
}

extern "C" int mofo_diff_attention_bwd(const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, int B, int Nq, int Nk, int H, int Hkv,
                                       float scale, const void* lam, int lam_heads, float lam_init, const void* gamma, int param_is_bf16, float eps,
                                       float out_scale, const int* kv_len, int causal, const void* o, const void* o2, const float* lse2, const void* dout,
                                       int lddo, void* dq, int lddq, void* dk, int lddk, void* dv, int lddv, void* dlam, void* dgamma, int grad_is_bf16,
                                       float* ws, long long ws_elems, void* stream) {
    int rc = check("mofo_diff_attention_bwd", q, ldq, k, ldk, v, ldv, B, Nq, Nk, H, Hkv, scale, lam, lam_heads, causal, gamma != nullptr, eps);
    if (rc) return rc;
    if (!o || !o2 || !lse2 || !dout || !dq || !dk || !dv || !dlam || !ws) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_bwd: null pointer");
    if (!gamma != !dgamma) MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_bwd: gamma and dgamma go together");
    if (lddo < H * HV || lddq < H * HV || lddk < Hkv * HV || lddv < Hkv * HV || (lddo | lddq | lddk | lddv) % 8)
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_diff_attention_bwd: bad leading dims of the gradients");
    if (lddo > (1 << 24)) MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_diff_attention_bwd: row pitch above 2^24");
    if (((uintptr_t)o | (uintptr_t)o2 | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15)
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_diff_attention_bwd: tensors must be 16-byte aligned");
    if (ws_elems < mofo_diff_attention_bwd_ws(B, Nq, Nk, H, Hkv, gamma != nullptr))
        MOFO_FAIL(MOFO_EINVAL, "mofo_diff_attention_bwd: ws of %lld floats is too small", ws_elems);
    {
        const long long HW = (long long)H * HV * 2, KW = (long long)Hkv * HV * 2, Mq = (long long)B * Nq, Mk = (long long)B * Nk, es = param_is_bf16 ? 2 : 4,
                        eg = grad_is_bf16 ? 2 : 4;
        const MofoSpan outs[] = {{"dq", dq, Mq, HW, 2LL * lddq}, {"dk", dk, Mk, KW, 2LL * lddk}, {"dv", dv, Mk, KW, 2LL * lddv}, {"dlam", dlam, 1, 256LL * lam_heads * eg, 0},
                                 {"dgamma", dgamma, 1, HV * eg, 0}, {"ws", ws, 1, mofo_diff_attention_bwd_ws(B, Nq, Nk, H, Hkv, gamma != nullptr) * 4, 0}};
        const MofoSpan in[] = {{"q", q, Mq, HW, 2LL * ldq}, {"k", k, Mk, KW, 2LL * ldk}, {"v", v, Mk, KW, 2LL * ldv}, {"lam", lam, 1, 256LL * lam_heads * es, 0},
                               {"gamma", gamma, 1, HV * es, 0}, {"kv_len", kv_len, 1, 4LL * B, 0}, {"o", o, 1, Mq * HW, 0}, {"o2", o2, 1, Mq * HW, 0},
                               {"lse2", lse2, 1, 8 * Mq * H, 0}, {"dout", dout, Mq, HW, 2LL * lddo}};
        MOFO_CHECK_APART("mofo_diff_attention_bwd", outs, 6, in, 10);
    }
    hipStream_t s = (hipStream_t)stream;
    const DiffArgs a = make_args(q, ldq, k, ldk, v, ldv, B, Nq, Nk, H, Hkv, scale, lam, lam_heads, lam_init, gamma, param_is_bf16, eps, out_scale, kv_len, causal);
    const size_t rows = (size_t)B * Nq * H;
    f32x4* stats = (f32x4*)ws;                            // then dO in bf16 (norm only), block partials, the heads' lambda
    bf16_t* d_o = (bf16_t*)(ws + rows * 4);
    float* part = ws + rows * 4 + (gamma ? rows * (HV / 2) : 0);
    float* lams = part + (size_t)H * row_blocks(B, Nq, H) * (HV + 1);
    const int nb = row_blocks(B, Nq, H);
    const bf16_t* dy = gamma ? d_o : (const bf16_t*)dout;
    const size_t lddy = gamma ? (size_t)H * HV : (size_t)lddo;
    const long long groups = (long long)B * Hkv, kt = (Nk + 31) / 32, qt = (long long)a.G * ((Nq + 31) / 32);
    bool q4 = four_way(groups, a.R, kt, causal == 1), k4 = four_way(groups, Nk, qt, causal != 0);
    Cut cut = {ceil_div(a.R, 128), 0.0};
    if (!causal && qt == kt) {                            // equal blocks throughout: dQ's last rows may fill up the last round
        // us, dK / dV and dQ in four-way blocks, and in 128-row blocks with a tail: 6 heads x 12544 2060 / 1822, 12 x 6000 975 / 846, 6 x 1568 65 / 76
        const long long nk = groups * ceil_div(Nk, 128), nq = groups * cut.nx, nq4 = groups * ceil_div(a.R, 32);
        const Cut c = cut_rows(nk, groups, a.R, kt);
        const double chosen = q4 && k4 ? block_time(true, groups * kt + nq4, kt, false)
                              : q4 || k4 ? block_time(k4, k4 ? groups * kt : nk, kt, false) + block_time(q4, q4 ? nq4 : nq, kt, false) : 1e30;
        if (1.15 * c.time < chosen) {                     // a step of dK / dV is longer than the model's
            q4 = k4 = false;
            cut = c;
        }
    }
    GradArgs g = {a, dy, lddy, stats, lams, part, (bf16_t*)dq, (bf16_t*)dk, (bf16_t*)dv, (size_t)lddq, (size_t)lddk, (size_t)lddv, dlam, dgamma, nb, grad_is_bf16};
    g.params = lam_heads + (dgamma ? 16 : 0);
    g.np = (g.params + 7) / 8 * 8;
    g.nxk = ceil_div(Nk, k4 ? 32 : 128);
    const long long nk_blocks = grid_of(a, g.nxk);
    g.nxq = q4 ? ceil_div(a.R, 32) : (int)cut.nx;
    g.spread = spread_of(a);
    const int tail = q4 ? 0 : tail_blocks(cut, a.R);
    const long long blocks = g.np + nk_blocks + grid_of(a, g.nxq);
    rc = check_blocks("mofo_diff_attention_bwd", std::max(blocks, grid_of(a, tail)));
    if (rc) return rc;
    g.nk = (int)nk_blocks;
    hipLaunchKernelGGL(diff_rows_kernel, dim3(nb, H), dim3(256), 0, s, a, (const bf16_t*)o, (const bf16_t*)o2, (const bf16_t*)dout, (size_t)lddo, lse2, d_o, stats, part, lams);
    MOFO_CHECK_LAUNCH("mofo_diff_attention_bwd(rows)");
    const dim3 grid((unsigned)blocks);
    if (q4 && k4) hipLaunchKernelGGL((diff_grad_kernel<true, true>), grid, dim3(256), 0, s, g);
    else if (q4) hipLaunchKernelGGL((diff_grad_kernel<true, false>), grid, dim3(256), 0, s, g);
    else if (k4) hipLaunchKernelGGL((diff_grad_kernel<false, true>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((diff_grad_kernel<false, false>), grid, dim3(256), 0, s, g);
    MOFO_CHECK_LAUNCH("mofo_diff_attention_bwd(gradients)");
    if (tail) {
        g.a.row0 = g.nxq * 128;
        g.np = g.params = g.nk = 0;
        g.nxq = tail;
        hipLaunchKernelGGL((diff_grad_kernel<true, false>), dim3((unsigned)grid_of(a, tail)), dim3(256), 0, s, g);
        MOFO_CHECK_LAUNCH("mofo_diff_attention_bwd(last rows)");
    }
    return MOFO_OK;
}
