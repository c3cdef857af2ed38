// Rotary positions over several axes (time, row, column) for gfx950: the first 2 * pairs columns of every head are pairs that turn by
// pos[axis] * freq[pair]; axis a owns sections[a] consecutive pairs.  With (c, s) = (cos, sin) of a pair's angle
//   (a, b) -> (a c - b s, a s + b c),
// the gradient is the same turn by the negative angle (INV).
//
// Angles: position x turns per position in 64 bits, the whole turns taken off there, cos / sin of the rest in f32 -- exact to f32 for
// any int32 position, where an f32 product is off by 1e-2 rad at position 1e5.  The angles of a token are the same for all its heads:
// a block takes up to ROPE_TOK tokens, puts their pairs' (cos, sin) into LDS once and turns all heads from there.
// HBM-bound: every element is read once and written once, 16 bytes a lane: 32 x 1568 tokens x 24 heads in bf16 57 us of graph time,
// 5.4 TB/s; below some thousand tokens it is the launch, 3 us of GPU time and 9 of the host's call.
#include "common.h"
#include "../../include/mofo_hip.h"

namespace {

constexpr int ROPE_MAX_PAIRS = 128;
constexpr int ROPE_TOK = 8;

struct RopeArgs {
    const void* x;
    void* out;
    size_t ldx, ldo;
    int M, heads, hd, pairs, tok_per_block;
    const double* freqs;      // [pairs] turns per position
    const int* pos;           // [M, naxes], or NULL: tok_idx names the place on a grid of (.., gh, gw)
    const int* tok_idx;       // [M]
    int naxes, end0, end1, end2, gh, gw;
    bool in_place;
};

template <bool BF>
__device__ __forceinline__ void load8(const void* p, size_t off, float* v) {
    if constexpr (BF) {
        const u32x4 w = *(const u32x4*)((const bf16_t*)p + off);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = bf16lo_to_f32(w[e]);
            v[2 * e + 1] = bf16hi_to_f32(w[e]);
        }
    } else {
        const f32x4 a = *(const f32x4*)((const float*)p + off), b = *(const f32x4*)((const float*)p + off + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    }
}

template <bool BF>
__device__ __forceinline__ void store8(void* p, size_t off, const float* v) {
    if constexpr (BF) {
        *(u32x4*)((bf16_t*)p + off) = u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    } else {
        *(f32x4*)((float*)p + off) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)((float*)p + off + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
}

template <bool BF, bool INTER, bool INV>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeArgs a) {
    __shared__ float2 cs[ROPE_TOK * ROPE_MAX_PAIRS];
    const int tid = threadIdx.x;
    const int m0 = blockIdx.x * a.tok_per_block;
    const int nt = a.M - m0 < a.tok_per_block ? a.M - m0 : a.tok_per_block;
    for (int idx = tid; idx < nt * a.pairs; idx += 256) {
        const int t = idx / a.pairs, i = idx - t * a.pairs;
        const int axis = (i >= a.end0) + (i >= a.end1) + (i >= a.end2);
        int p;
        if (a.pos) {
            p = a.pos[(size_t)(m0 + t) * a.naxes + axis];
        } else {
            const int id = a.tok_idx[m0 + t], plane = a.gh * a.gw;
            const int in = id % plane;
            p = axis == 0 ? id / plane : axis == 1 ? in / a.gw : in % a.gw;
        }
        double turns = (double)p * a.freqs[i];
        turns -= rint(turns);
        float s, c;
        sincospif(2.0f * (float)turns, &s, &c);
        cs[idx] = float2{c, INV ? -s : s};
    }
    __syncthreads();
    // items of 16 columns: eight pairs, or a run of columns that no pair covers (copied)
    const int per_head = a.hd >> 4, per_tok = per_head * a.heads, octets = a.pairs >> 3;
    for (int it = tid; it < nt * per_tok; it += 256) {
        const int t = it / per_tok, r = it - t * per_tok;
        const int h = r / per_head, j = r - h * per_head;
        const size_t xo = (size_t)(m0 + t) * a.ldx + h * a.hd, oo = (size_t)(m0 + t) * a.ldo + h * a.hd;
        const bool pairs_here = j < octets;
        if (!pairs_here && a.in_place) continue;
        const int lo = INTER || !pairs_here ? 16 * j : 8 * j;
        const int hi = INTER || !pairs_here ? 16 * j + 8 : a.pairs + 8 * j;
        float u[8], v[8];
        load8<BF>(a.x, xo + lo, u);
        load8<BF>(a.x, xo + hi, v);
        if (pairs_here) {
            const float2* w = cs + t * a.pairs + 8 * j;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 z = w[e];
                float& p = INTER ? (e < 4 ? u[2 * e] : v[2 * e - 8]) : u[e];
                float& q = INTER ? (e < 4 ? u[2 * e + 1] : v[2 * e - 7]) : v[e];
                const float pn = p * z.x - q * z.y;
                q = p * z.y + q * z.x;
                p = pn;
            }
        }
        store8<BF>(a.out, oo + lo, u);
        store8<BF>(a.out, oo + hi, v);
    }
}

template <bool BF, bool INTER>
void launch(const RopeArgs& a, int inverse, hipStream_t s) {
    const dim3 grid((unsigned)(((long long)a.M + a.tok_per_block - 1) / a.tok_per_block));
    if (inverse) hipLaunchKernelGGL((rope_axes_kernel<BF, INTER, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_axes_kernel<BF, INTER, false>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" int mofo_rope_axes(const void* x, int x_is_bf16, int ldx, void* out, int ldo, int M, int heads, int head_dim, const double* freqs,
                              int naxes, const int* sections, const int* pos, const int* tok_idx, int grid_h, int grid_w, int interleaved,
                              int inverse, void* stream) {
    if (!x || !out || !freqs || !sections) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: null pointer");
    if (M <= 0 || heads <= 0 || head_dim <= 0) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: bad dims M=%d heads=%d head_dim=%d", M, heads, head_dim);
    if (naxes < 1 || naxes > 4) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: naxes=%d must be 1..4", naxes);
    int end[4] = {1 << 30, 1 << 30, 1 << 30, 1 << 30};
    long long pairs = 0;
    for (int k = 0; k < naxes; ++k) {
        if (sections[k] < 0 || sections[k] > ROPE_MAX_PAIRS) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: sections[%d]=%d", k, sections[k]);
        pairs += sections[k];
        if (k + 1 < naxes) end[k] = (int)pairs;
    }
    if (head_dim % 16 || head_dim > 1024 || pairs < 8 || pairs % 8 || pairs > ROPE_MAX_PAIRS || 2 * pairs > head_dim)
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_rope_axes: %lld pairs in heads of %d: pairs a multiple of 8 up to %d, 2 * pairs <= head_dim, head_dim a multiple of 16 up to 1024",
                  pairs, head_dim, ROPE_MAX_PAIRS);
    if (!pos == !tok_idx) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: exactly one of pos and tok_idx");
    if (tok_idx && (naxes != 3 || grid_h <= 0 || grid_w <= 0 || (long long)grid_h * grid_w > 0x7fffffffLL))
        MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: tok_idx needs three axes and a grid (got naxes=%d, %d x %d)", naxes, grid_h, grid_w);
    const long long W = (long long)heads * head_dim;
    const int vec = x_is_bf16 ? 8 : 4;
    if (ldx < W || ldo < W || ldx % vec || ldo % vec || ((uintptr_t)x & 15) || ((uintptr_t)out & 15))
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_rope_axes: rows of 16-byte aligned pieces (ldx=%d, ldo=%d for %lld columns)", ldx, ldo, W);
    if (x == out && ldx != ldo) MOFO_FAIL(MOFO_EINVAL, "mofo_rope_axes: in place with two row pitches (%d, %d)", ldx, ldo);
    {
        const int es = x_is_bf16 ? 2 : 4;
        const MofoSpan o = {"out", out, M, W * es, (long long)ldo * es};
        const MofoSpan in[] = {{"x", x == out ? nullptr : x, M, W * es, (long long)ldx * es}, {"freqs", freqs, 1, pairs * 8, 0},
                               {"pos", pos, 1, (long long)M * naxes * 4, 0}, {"tok_idx", tok_idx, 1, (long long)M * 4, 0}};
        MOFO_CHECK_APART("mofo_rope_axes", &o, 1, in, 4);
    }
    // few tokens: one a block, to fill the card (160 tokens x 24 heads in bf16, us by tokens a block: 1 3.1, 4 3.7, 8 4.2; 2048 4.5, 4.6, 5.0);
    // many: several, for the angles' share of a block's time (8192 12.4, 9.7, 9.8; 50176 76, 57, 58), more of them if their rows are short
    // (50176 x 3 heads 39, 15, 13; 14997 x 7 heads in f32: 4 11.7, 8 11.2)
    const int tok_per_block = M < 2048 ? 1 : W * (x_is_bf16 ? 2 : 4) >= 2048 ? ROPE_TOK / 2 : ROPE_TOK;
    const long long blocks = ((long long)M + tok_per_block - 1) / tok_per_block;
    if (blocks > MOFO_MAX_BLOCKS_256)
        MOFO_FAIL(MOFO_EUNSUPPORTED, "mofo_rope_axes: M=%d takes %lld blocks of %d rows (at most %lld)", M, blocks, tok_per_block, MOFO_MAX_BLOCKS_256);
    RopeArgs a;
    a.x = x;
    a.out = out;
    a.ldx = (size_t)ldx;
    a.ldo = (size_t)ldo;
    a.M = M;
    a.heads = heads;
    a.hd = head_dim;
    a.pairs = (int)pairs;
    a.freqs = freqs;
    a.pos = pos;
    a.tok_idx = tok_idx;
    a.naxes = naxes;
    a.end0 = end[0];
    a.end1 = end[1];
    a.end2 = end[2];
    a.gh = grid_h;
    a.gw = grid_w;
    a.in_place = x == out;
    a.tok_per_block = tok_per_block;
    hipStream_t s = (hipStream_t)stream;
    if (x_is_bf16) {
        if (interleaved) launch<true, true>(a, inverse, s);
        else launch<true, false>(a, inverse, s);
    } else {
        if (interleaved) launch<false, true>(a, inverse, s);
        else launch<false, false>(a, inverse, s);
    }
    MOFO_CHECK_LAUNCH("mofo_rope_axes");
    return MOFO_OK;
}
