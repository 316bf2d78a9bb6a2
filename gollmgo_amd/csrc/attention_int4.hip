// attention_int4.hip — the MFMA attention kernel of 4-bit pools: head_dim 64 or 128, 16-token blocks.
//
// A 256-thread workgroup takes one piece of an item (a sequence, a kv head and up to 16 * NT of its
// G * R query rows): the plan's pieces as in attention_mfma.h, or the whole item where nothing would
// be cut. Its four waves stream disjoint chunks of 64 or 32 tokens (int4_chunk_tokens) and merge at the
// end. Lane = 16 * g4 + c16. Below, chunks of 64 (four blocks).
//
// Mathematics. A token's key is s_k (n - z_k) and its value s_v (m - z_v), n and m whole 0..15.
//   score     = s_k (sum q n - z_k sum q): the products run over the codes alone. The zero point is
//               one more step of the contraction: operand (z, z) against (-sum q) in two f16 parts.
//   P.V       = sum p s_v m - sum p s_v z_v: p s_v is the A operand, the codes and, as one more
//               column tile, the zero points are B operands; the difference is taken at the end. Both sums
//               grow with the keys where their difference averages out, so each half of the dims has zero
//               points in the units of its codes (columns 0..7: z, 8..15: 16 z): what the matrix unit cuts
//               off the products is then alike in both and leaves with the difference (f16 outputs over 200 000 keys:
//               8.0e-4 off in norm with one column for both halves, 2.4e-4 so, their own rounding 2.1e-4).
// Codes go into the f16 operands without a conversion: the bits 0..15 (or 16 times that, the upper
// half of a byte left in place) are the f16 subnormals n * 2^-24 (n * 2^-20), which
// v_mfma_f32_16x16x32_f16 takes exactly. Eight codes cost one shift and four ands (an or with 0x6400
// and a subtraction per pair would make it nine), the power of two goes into the score's multiplier,
// and the 16 of every other operand pair into the queries (K) or the column tile (V).
//   S^T = K . Q^T : lane holds token 4 * (c16 / 4) + ... of its S tile as the A row, dims of lane group
//               g4 as k. A K row is head_dim / 2 bytes, its lane group's run one 16- or 8-byte load.
//               The result gives lane (g4, c16) row c16 and the 16 tokens of block g4.
//   O += P . V  : those 16 tokens are the A operand as they are; the V tile [D/2][16] gives a lane 16
//               tokens of dims i and i + D/2 in one 16-byte load, two column tiles.
// Each token's scales and zero points are one word. A lane loads and decodes one token's and puts them
// into LDS, from where every lane takes its sixteen (decoded by their readers they cost 100
// instructions a chunk).
//
// p s_v is held in f16 in units of B 2^-10, B a power of two at or above every s_v the wave has seen
// (O is rescaled when it grows). Values whose scales lie up to 2^12 apart keep 11 bits down to
// p = 2^-12 that way, and half a step of 2^-35 B below; a piece whose scales lie further apart is
// computed row by row in fp32. Each query row has a power of two of its own (its largest |q| in
// [2^7, 2^8)), so rows do not touch.
// PREC (fp32 queries or outputs): queries and p s_v in two f16 parts each, 22 bits, and the codes less
// their zero points as normal f16 numbers in the operands (exact). Two roundings that f16 probabilities
// hide would show in fp32 results: codes and zero points summed apart leave 2^-20 of the row's range, and
// the matrix unit aligns a subnormal's products by the exponent it is stored with, up to ten bits above
// them, so that the sums keep about 17 bits (2-norm errors against 64 bits, 24
// and 12 rows over 230 and 20 keys: 1.7e-5 and 1.3e-5 with subnormals, 4.5e-7 and 2.3e-7 with these).
// Subtracting is 64 + 16 * 4 instructions more a chunk.
//
// Bound: one read of a token's 2 * (D / 2) + 4 bytes serves all its kv head's rows. Planned calls, 8 kv
// heads of 128, bf16, kernel time: 64 sequences of 1024-8192 keys, 24 rows a head (two row tiles),
// 346 MB 72 µs, 4.8 TB/s (the same loads with nothing done to them 5.0 over the whole call); 128
// sequences of 256-2048 keys, four rows 29.3 µs, 5.2 TB/s. Memory, both. 8 sequences of 16384-32768
// keys, 36 rows (three row tiles) 77 µs, 2.8 TB/s: per SIMD 39 µs of vector and 19 of matrix
// instructions, two waves to overlap them. One sequence of 3006 keys, 20 rows 17 µs: a chain of round
// trips (table, block ids, keys and values, the pieces' records).
#include "attention_mfma.h"
#include "lanes.h"

namespace gg {
namespace {

constexpr float kI4Spread = 4096.f;       // ratio of value scales that f16 probabilities take
// A row's maximum moves only when a chunk exceeds it by 2^kI4Slack: exponentials up to 2^5 are as good
// as up to 1, and O, which every new maximum would rescale (with sixteen rows to a wave, nearly every
// chunk finds one), is left alone.
constexpr float kI4Slack = 5.f;
constexpr float kI4Unit = 1024.f;         // p s_v in units of B / kI4Unit: at most 2^15
constexpr uint32_t kLoNib = 0x000f000fu, kHiNib = 0x00f000f0u;
template <bool PREC>
constexpr int kCodeExp = PREC ? 0 : 24;   // a code stands in its operand as n 2^-kCodeExp

// Eight codes of a K dword as an MFMA operand: (n0, n4), 16 (n1, n5), (n2, n6), 16 (n3, n7), of each pair
// `base` more.
__device__ __forceinline__ uint4 k_operand8(uint32_t w, uint32_t base) {
    const uint32_t u = w >> 8;
    return make_uint4((w & kLoNib) | base, (w & kHiNib) | base, (u & kLoNib) | base, (u & kHiNib) | base);
}

__device__ __forceinline__ uint32_t pk_sub_f16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) - __builtin_bit_cast(f16x2, b));
}
// PREC: codes and zero points as 1024 + n (f16 holds whole numbers there), whose difference is exact.
constexpr uint32_t kF16_1024 = 0x64006400u;
// An operand's codes less their zero points: z for the first and third pair, 16 z for the others.
__device__ __forceinline__ uint4 less_zero(uint4 v, uint32_t z0, uint32_t z1, uint32_t z2, uint32_t z3) {
    return make_uint4(pk_sub_f16(v.x, z0), pk_sub_f16(v.y, z1), pk_sub_f16(v.z, z2), pk_sub_f16(v.w, z3));
}

__device__ __forceinline__ uint32_t f16_pair(float a, float b) { return cvt_pk_f16(a, b); }

template <int NT, int HD, bool PREC, int TOK>
struct Int4Shared {
    static constexpr int kTok = TOK;
    static constexpr int kMM = HD / 32, kParts = PREC ? 2 : 1;
    uint4 q[kParts][NT][kMM][64];   // B operands of S
    uint32_t qz[NT * 16];           // -sum q of a row, two f16 parts
    float qmul[NT * 16];            // the row's score multiplier, log2 domain
    // The chunk's tokens, decoded by the lane that loaded each token's word.
    float ks[kWaves][kTok], vs[kWaves][kTok];
    uint32_t kz[kWaves][kTok];                       // (z, z)
    __align__(16) uint16_t vz[kWaves][kParts == 1 ? 2 : 1][kTok];  // in the order of the V operands: z, 16 z
    float m[kWaves][NT * 16], l[kWaves][NT * 16];
    int bad[kWaves];
    __align__(16) float o[kWaves][16][HD + 4];
};

// Row `row` of the piece by the per-row kernel's steps, for pieces whose value scales are too far apart.
template <int HD>
__device__ __forceinline__ void int4_piece_by_rows(const AttnArgs& a, const KVView& kv, const PieceDesc& d, int rows,
                                                   int rec_rows, float* s_row) {
    constexpr int kDC = HD / 64;
    const int G = a.num_q_heads / kv.Hkv, lane = threadIdx.x & 63;
    float* s_q = s_row;
    float* s_p = s_row + HD;
    size_t* s_vrow = (size_t*)(s_row + HD + 64);
    for (int r = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); r < rows; r += kWaves) {
        const int j = (d.row0 + r) / G, g = (d.row0 + r) % G;
        const size_t obase = (((size_t)d.b * a.rows + j) * a.num_q_heads + (size_t)d.kvh * G + g) * HD;
        __builtin_amdgcn_wave_barrier();  // (the previous row's reads)
#pragma unroll
        for (int c = 0; c < kDC; ++c) s_q[lane + 64 * c] = load_as_f32(a.q, a.q_dtype, obase + lane + 64 * c);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float acc[kDC], m, l;
        generic_partition<GG_DTYPE_INT4, kDC, true>(a, kv, d.b, d.kvh, d.t0, min(d.t_end, d.ctx - d.nrows + j + 1), s_q, s_p,
                                                     s_vrow, acc, m, l);
        if (d.rec < 0) {
            const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
            for (int c = 0; c < kDC; ++c) store_from_f32(a.out, a.out_dtype, obase + lane + 64 * c, acc[c] * inv);
        } else {
            const size_t q = (size_t)d.rec * rec_rows + r;
#pragma unroll
            for (int c = 0; c < kDC; ++c) store_agent(a.ws_acc + q * HD + lane + 64 * c, acc[c]);
            if (lane == 0) store_agent2(a.ws_ml + q * 2, m, l);
        }
    }
}

// The piece's queries: HD / 8 threads a row, eight dims (one K dword) each. Loaded before the piece's
// keys and values (loads retire in order, so the staging then waits for these alone), and put into
// LDS as MFMA operands, scaled row by row.
template <int NT, int HD, bool PREC, int TOK>
struct Int4Queries {
    static constexpr int kPer = HD / 8, kStep = 256 / kPer, kIt = (16 * NT + kStep - 1) / kStep;
    uint4 w[kIt][PREC ? 2 : 1];

    __device__ __forceinline__ void load(const AttnArgs& a, const KVView& kv, const PieceDesc& d, int rows) {
        const int G = a.num_q_heads / kv.Hkv;
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
            const int r = min((int)threadIdx.x / kPer + it * kStep, rows - 1);
            const int j = (d.row0 + r) / G, g = (d.row0 + r) % G;
            const size_t at = (((size_t)d.b * a.rows + j) * a.num_q_heads + (size_t)d.kvh * G + g) * HD + 8 * (threadIdx.x % kPer);
            struct __attribute__((packed, aligned(2))) U4 { uint4 v; };
            if (PREC && a.q_dtype == GG_DTYPE_F32) {
                struct __attribute__((packed, aligned(4))) F4 { uint4 v; };
                w[it][0] = ((const F4*)((const float*)a.q + at))[0].v;
                w[it][PREC ? 1 : 0] = ((const F4*)((const float*)a.q + at))[1].v;
            } else {
                w[it][0] = ((const U4*)((const uint16_t*)a.q + at))->v;
            }
        }
    }

    __device__ __forceinline__ void stage(const AttnArgs& a, int rows, Int4Shared<NT, HD, PREC, TOK>& s) const {
        constexpr int kMM = HD / 32;
        const int ch = threadIdx.x % kPer;
#pragma unroll
        for (int it = 0; it < kIt; ++it) {
            const int r = threadIdx.x / kPer + it * kStep;
            if (r >= 16 * NT) break;
            float f[8];
            const uint32_t x[4] = {w[it][0].x, w[it][0].y, w[it][0].z, w[it][0].w};
            if (PREC && a.q_dtype == GG_DTYPE_F32) {
                const uint4 y = w[it][PREC ? 1 : 0];
                f[0] = __uint_as_float(x[0]), f[1] = __uint_as_float(x[1]), f[2] = __uint_as_float(x[2]), f[3] = __uint_as_float(x[3]);
                f[4] = __uint_as_float(y.x), f[5] = __uint_as_float(y.y), f[6] = __uint_as_float(y.z), f[7] = __uint_as_float(y.w);
            } else if (a.q_dtype == GG_DTYPE_BF16) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = f16_bits_to_f32((uint16_t)(x[e >> 1] >> (16 * (e & 1))));
            }
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = r < rows ? f[e] : 0.f;
                mx = fmaxf(mx, fabsf(f[e]));  // (a NaN is passed over)
            }
            mx = group_max<kPer>(mx);
            int e2 = 8;
            if (mx > 0.f && mx <= 3.402823466e38f) (void)frexpf(mx, &e2);
            const int k = e2 - 8;
            // Two factors: 2^-k alone may overflow.
            const float s1 = ldexpf(1.f, -(k / 2)), s2 = ldexpf(1.f, -(k - k / 2));
            // Operand order (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16.
            float sum = 0.f;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float down = p & 1 ? 0.0625f : 1.f, up = p & 1 ? 16.f : 1.f;
                const float u = f[p] * s1 * s2 * down, v = f[p + 4] * s1 * s2 * down;
                hi[p] = f16_pair(u, v);
                const float hu = f16_bits_to_f32((uint16_t)hi[p]), hv = f16_bits_to_f32((uint16_t)(hi[p] >> 16));
                sum += (hu + hv) * up;
                if constexpr (PREC) lo[p] = f16_pair(u - hu, v - hv);
            }
            const int slot = 16 * (ch / kMM) + (r & 15);
            s.q[0][r >> 4][ch % kMM][slot] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PREC) s.q[1][r >> 4][ch % kMM][slot] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            sum = group_sum<kPer>(sum);
            if (ch == 0) {
                const float top = f16_bits_to_f32(f32_to_f16_bits(-sum));
                s.qz[r] = f16_pair(top, -sum - top);
                // (Positive and finite: a hidden score times it stays -inf.)
                const float mul = ldexpf(a.scale * kLog2e, k + kCodeExp<PREC>);
                s.qmul[r] = fminf(fmaxf(mul, 0x1p-126f), 3.0e38f);
            }
        }
    }
};

template <int NT, int HD, bool PREC, int TOK>
__device__ __forceinline__ void int4_piece(const AttnArgs& a, const KVView& kv, const PieceDesc& d) {
    constexpr int kTok = TOK, kNS = kTok / 16, kN = 4 * kNS;  // a chunk's tokens, S tiles; a lane's tokens
    using IO = PieceIO<GG_DTYPE_INT8, kTok, HD>;    // (block ids of chunks)
    using Geom = Geo<1, kTok, HD>;                  // (tokens of lanes and S tiles)
    constexpr int kMM = HD / 32, kVT = HD / 32;     // K operands of a token; V loads of a lane
    constexpr int kParts = PREC ? 2 : 1;
    constexpr int kKW = HD / 32;                    // dwords of a lane's K run
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g4 = lane >> 4;
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);
    const int G = a.num_q_heads / kv.Hkv;
    const int ctx = d.ctx, nrows = d.nrows;
    if (nrows <= 0 || nrows > ctx) return;
    const int rows = min(G * nrows - d.row0, 16 * NT);
    if (rows <= 0) return;
    const int first_masked = ctx - nrows;
    const int nchunks = (d.t_end - d.t0 + kTok - 1) / kTok;
    __shared__ Int4Shared<NT, HD, PREC, TOK> s;

    // The call's own rows in this piece: written first, by the whole workgroup. (Row groups write
    // the same bytes.)
    if (a.k_new) {
        const int j0 = max(0, d.t0 - first_masked), j1 = min(nrows, d.t_end - first_masked);
        if (j0 < j1) {
            append_int4_rows(a, kv, d.b, d.kvh, ctx, nrows, j0, j1);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __syncthreads();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        }
    }

    // The lane's first token in the chunk (its P run); the token it decodes the scales of; its K rows.
    const int run = 16 * Geom::bq(g4) + Geom::ob(g4);
    const int own = run + (c16 & (kN - 1));
    const int krow = 16 * Geom::bq(c16 >> 2) + Geom::ob(c16 >> 2) + (c16 & 3);  // of S tile 0; 4 t further of tile t
    uint32_t kr[kNS][kKW];        // K: S tile t, the lane's token of it
    uint32_t vr[kVT][kN / 4];     // V: the lane's tokens, dims 16 i + c16 and that plus HD / 2
    uint32_t wr;                  // word of token `own`
    auto load_k = [&](const LaneBlocks bl) {
        const int blk = max(bl.k, 0);
        const uint8_t* p = kv.kc + ((size_t)blk * kv.Hkv + d.kvh) * (size_t)(kBS * HD) + (size_t)(krow & 15) * (HD / 2) + 4 * kKW * g4;
#pragma unroll
        for (int t = 0; t < kNS; ++t) {
            if constexpr (kKW == 4) {
                const uint4 x = *(const uint4*)(p + t * 4 * (HD / 2));
                kr[t][0] = x.x, kr[t][1] = x.y, kr[t][2] = x.z, kr[t][3] = x.w;
            } else {
                const uint2 x = *(const uint2*)(p + t * 4 * (HD / 2));
                kr[t][0] = x.x, kr[t][1] = x.y;
            }
        }
    };
    auto load_word = [&](const LaneBlocks bl) {
        wr = kv.words[((size_t)max(bl.v, 0) * kv.Hkv + d.kvh) * kBS + (own & 15)];
    };
    auto load_v = [&](const LaneBlocks bl) {
        const uint8_t* p = kv.vc + ((size_t)max(bl.v, 0) * kv.Hkv + d.kvh) * (size_t)(kBS * HD) + (size_t)c16 * kBS + Geom::ob(g4);
#pragma unroll
        for (int i = 0; i < kVT; ++i) {
            if constexpr (kN == 16) {
                const uint4 x = *(const uint4*)(p + i * 16 * kBS);
                vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
            } else {
                const uint2 x = *(const uint2*)(p + i * 16 * kBS);
                vr[i][0] = x.x, vr[i][1] = x.y;
            }
        }
    };
    Int4Queries<NT, HD, PREC, TOK> qs;
    const auto fb = IO::first_blocks(a, d);
    qs.load(a, kv, d, rows);
    LaneBlocks bl_cur = IO::lane_blocks(kv, fb.r0, d.t_end), bl_next = IO::lane_blocks(kv, fb.r1, d.t_end);
    load_k(bl_cur);
    load_word(bl_cur);
    load_v(bl_cur);

    qs.stage(a, rows, s);
    __syncthreads();

    uint32_t qz[NT];
    float qmul[NT];
    int row_pos[NT];  // last key that row c16 sees
#pragma unroll
    for (int rt = 0; rt < NT; ++rt) {
        const int r = rt * 16 + c16;
        qz[rt] = g4 == 0 ? s.qz[r] : 0u;  // k = 0, 1 of the contraction: lane group 0
        qmul[rt] = s.qmul[r];
        row_pos[rt] = r < rows ? first_masked + (d.row0 + r) / G : ctx - 1;
    }

    f32x4 o[NT][2 * kVT], oz[NT];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int rt = 0; rt < NT; ++rt) {
        m_run[rt] = -1e30f;
        l_run[rt] = 0.f;
        oz[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2 * kVT; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float bound = 0.f, vnorm = 0.f;   // B, and kI4Unit / B (wave-uniform)
    // Token `own` in the V operands: of each eight, tokens (0, 2), (1, 3), (4, 6), (5, 7).
    const int vz_at = (own & ~7) + (own & 4) + 2 * (own & 1) + ((own >> 1) & 1);
    float vs_min = 3.0e38f;           // smallest value scale of the lane's tokens

    for (int ch = wave_u; ch < nchunks; ch += kWaves) {
        const int tc = d.t0 + ch * kTok;
        const int tlane = tc + run;
        const bool missing = bl_cur.v < 0;

        // The chunk's scales and zero points to LDS (this wave's own slots: its LDS operations run in
        // order). Tokens behind the end and in missing blocks count as values of scale 0.
        {
            const bool live = !missing && tc + own < ctx;
            const float vs = live ? int4_v_scale(wr) : 0.f;
            vs_min = vs > 0.f ? fminf(vs_min, vs) : vs_min;
            if (__builtin_expect(__any(vs > bound), 0)) {
                // Value scales past B: B grows, and what has been summed shrinks with it.
                const float top = wave_max(vs);
                const float grown = __uint_as_float((__float_as_uint(top) + 0x7fffffu) & 0x7f800000u);
                const float f = __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(bound / grown)));
                bound = __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(grown)));
                vnorm = kI4Unit / bound;
#pragma unroll
                for (int rt = 0; rt < NT; ++rt) {
                    oz[rt] *= f;
#pragma unroll
                    for (int t = 0; t < 2 * kVT; ++t) o[rt][t] *= f;
                }
            }
            __builtin_amdgcn_wave_barrier();
            const uint32_t zk = wr & 15u;
            s.ks[wave][own] = int4_k_scale(wr);
            s.vs[wave][own] = vs * vnorm;
            s.kz[wave][own] = zk | (zk << 16);
            s.vz[wave][0][vz_at] = (uint16_t)int4_v_zero(wr);
            if constexpr (!PREC) s.vz[wave][1][vz_at] = (uint16_t)(int4_v_zero(wr) << 4);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }

        const typename IO::RawBlocks raw_after = IO::fetch_blocks(a, d.b, d.t0, ch + 2 * kWaves);
        const bool need_mask = tc + kTok - 1 >= first_masked || __any(missing);
        // ---- S^T = K . Q^T ----
        // (The Q index is opaque, so that the LDS reads stay in the loop.)
        int qlane;
        asm("" : "=v"(qlane) : "0"(lane), "s"(ch));
        f32x4 sacc[NT][kNS];
#pragma unroll
        for (int rt = 0; rt < NT; ++rt)
#pragma unroll
            for (int t = 0; t < kNS; ++t) sacc[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t kz[kNS];  // zero point of the lane's token of S tile t, a pair
#pragma unroll
        for (int t = 0; t < kNS; ++t) kz[t] = s.kz[wave][krow + 4 * t];
#pragma unroll
        for (int mm = 0; mm < kMM; ++mm) {
            uint4 qop[kParts][NT];
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int rt = 0; rt < NT; ++rt) qop[p][rt] = s.q[p][rt][mm][qlane];
#pragma unroll
            for (int t = 0; t < kNS; ++t) {
                uint4 kop = k_operand8(kr[t][mm], PREC ? kF16_1024 : 0u);
                if constexpr (PREC) {
                    const uint32_t z0 = kz[t] | kF16_1024, z1 = (kz[t] << 4) | kF16_1024;
                    kop = less_zero(kop, z0, z1, z0, z1);
                }
#pragma unroll
                for (int rt = 0; rt < NT; ++rt)
#pragma unroll
                    for (int p = 0; p < kParts; ++p) sacc[rt][t] = mfma(kop, qop[p][rt], sacc[rt][t], false);
            }
        }
        if constexpr (!PREC) {
#pragma unroll
            for (int t = 0; t < kNS; ++t)
#pragma unroll
                for (int rt = 0; rt < NT; ++rt)
                    sacc[rt][t] = mfma(make_uint4(kz[t], 0u, 0u, 0u), make_uint4(qz[rt], 0u, 0u, 0u), sacc[rt][t], false);
        }
        load_k(bl_next);
        load_word(bl_next);

        // ---- online softmax ----
        uint32_t pop[NT][kParts][kN / 2];
        float ks[kN], vs[kN];  // of the lane's tokens
#pragma unroll
        for (int t = 0; t < kNS; ++t) {
            const int at = run + 4 * t;
            const float4 x = *(const float4*)&s.ks[wave][at], y = *(const float4*)&s.vs[wave][at];
            ks[4 * t] = x.x, ks[4 * t + 1] = x.y, ks[4 * t + 2] = x.z, ks[4 * t + 3] = x.w;
            vs[4 * t] = y.x, vs[4 * t + 1] = y.y, vs[4 * t + 2] = y.z, vs[4 * t + 3] = y.w;
        }
#pragma unroll
        for (int rt = 0; rt < NT; ++rt) {
            float sc[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) sc[i] = sacc[rt][i >> 2][i & 3] * ks[i];
            if (__builtin_expect(need_mask, 0)) {
#pragma unroll
                for (int i = 0; i < kN; ++i) sc[i] = !missing && tlane + i <= row_pos[rt] ? sc[i] : -INFINITY;
            }
            float cmax = sc[0];
#pragma unroll
            for (int i = 1; i < kN; ++i) cmax = fmaxf(cmax, sc[i]);
            cmax *= qmul[rt];
            // (The row's maximum over its four lanes is taken only where one of them is past the slack.)
            if (__any(cmax > m_run[rt] + kI4Slack)) {
                cmax = max_over_rows(cmax);
                const float m_new = cmax > m_run[rt] + kI4Slack ? cmax : m_run[rt];
                const float alpha = __builtin_amdgcn_exp2f(m_run[rt] - m_new);
                l_run[rt] *= alpha;
                m_run[rt] = m_new;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float al = __shfl(alpha, 4 * g4 + i);
                    oz[rt][i] *= al;
#pragma unroll
                    for (int t = 0; t < 2 * kVT; ++t) o[rt][t][i] *= al;
                }
            }
            float psum = 0.f;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], qmul[rt], -m_run[rt]));
                psum += sc[i];
                sc[i] *= vs[i];
            }
            l_run[rt] += psum;
            // Operand order of a V dword: tokens (0, 2), (1, 3).
#pragma unroll
            for (int q = 0; q < kNS; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = sc[4 * q + e], y = sc[4 * q + e + 2];
                    const uint32_t h = f16_pair(x, y);
                    pop[rt][0][2 * q + e] = h;
                    if constexpr (PREC)
                        pop[rt][1][2 * q + e] =
                            f16_pair(x - f16_bits_to_f32((uint16_t)h), y - f16_bits_to_f32((uint16_t)(h >> 16)));
                }
        }

        // ---- O += P . V, the zero points as one more column tile ----
#pragma unroll
        for (int half = 0; half < kNS / 2; ++half) {
            const uint4 z = *(const uint4*)&s.vz[wave][PREC ? 0 : c16 >> 3][run + 8 * half];
            uint4 pa[NT][kParts];
#pragma unroll
            for (int rt = 0; rt < NT; ++rt)
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    const uint32_t* q = pop[rt][p] + 4 * half;
                    pa[rt][p] = make_uint4(q[0], q[1], q[2], q[3]);
                }
            if constexpr (!PREC) {
#pragma unroll
                for (int rt = 0; rt < NT; ++rt) oz[rt] = mfma(pa[rt][0], z, oz[rt], false);
            }
#pragma unroll
            for (int i = 0; i < kVT; ++i) {
                const uint32_t x = vr[i][2 * half], y = vr[i][2 * half + 1], x8 = x >> 8, y8 = y >> 8;
                constexpr uint32_t b = PREC ? kF16_1024 : 0u;
                uint4 lo = make_uint4((x & kLoNib) | b, (x8 & kLoNib) | b, (y & kLoNib) | b, (y8 & kLoNib) | b);
                uint4 hi = make_uint4((x & kHiNib) | b, (x8 & kHiNib) | b, (y & kHiNib) | b, (y8 & kHiNib) | b);
                if constexpr (PREC) {
                    lo = less_zero(lo, z.x | b, z.y | b, z.z | b, z.w | b);
                    hi = less_zero(hi, (z.x << 4) | b, (z.y << 4) | b, (z.z << 4) | b, (z.w << 4) | b);
                }
#pragma unroll
                for (int rt = 0; rt < NT; ++rt)
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        o[rt][i] = mfma(pa[rt][p], lo, o[rt][i], false);
                        o[rt][i + kVT] = mfma(pa[rt][p], hi, o[rt][i + kVT], false);
                    }
            }
        }
        load_v(bl_next);
        bl_cur = bl_next;
        bl_next = IO::lane_blocks(kv, raw_after, d.t_end);
    }

    // ---- merge the four waves ----
#pragma unroll
    for (int rt = 0; rt < NT; ++rt) {
        float lt = l_run[rt];
        lt += __shfl_xor(lt, 16);
        lt += __shfl_xor(lt, 32);
        if (g4 == 0) {
            s.m[wave][rt * 16 + c16] = m_run[rt];
            s.l[wave][rt * 16 + c16] = lt;
        }
    }
    const float lowest = wave_min(vs_min);
    if (lane == 0) s.bad[wave] = bound > kI4Spread * lowest;
    __syncthreads();
    if (__builtin_expect(s.bad[0] | s.bad[1] | s.bad[2] | s.bad[3], 0)) {
        int4_piece_by_rows<HD>(a, kv, d, rows, 16 * NT, &s.o[wave][0][0]);
        return;
    }
    const float unit = bound * ((float)(1 << kCodeExp<PREC>) / kI4Unit);
    for (int rt = 0; rt < NT; ++rt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rr = 4 * g4 + i, r = rt * 16 + rr;
            if (r >= rows) break;
            float mx = s.m[0][r];
#pragma unroll
            for (int u = 1; u < kWaves; ++u) mx = fmaxf(mx, s.m[u][r]);
            const float f = __builtin_amdgcn_exp2f(s.m[wave][r] - mx) * unit;
            const float oz_other = dpp<0x128>(oz[rt][i]);  // row_ror:8
            const float oz0 = c16 < 8 ? oz[rt][i] : oz_other, oz1 = c16 < 8 ? oz_other : oz[rt][i];
#pragma unroll
            for (int t = 0; t < kVT; ++t) {
                s.o[wave][rr][t * 16 + c16] = (o[rt][t][i] - oz0) * f;
                s.o[wave][rr][HD / 2 + t * 16 + c16] = (o[rt][t + kVT][i] - oz1) * (0.0625f * f);
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = threadIdx.x; e < 16 * (HD / 4); e += 256) {
            const int rr = e / (HD / 4), dim = 4 * (e % (HD / 4)), r = rt * 16 + rr;
            if (r >= rows) continue;
            float mx = s.m[0][r];
#pragma unroll
            for (int u = 1; u < kWaves; ++u) mx = fmaxf(mx, s.m[u][r]);
            float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < kWaves; ++u) {
                L += s.l[u][r] * __builtin_amdgcn_exp2f(s.m[u][r] - mx);
                const float4 v = *(const float4*)&s.o[u][rr][dim];
                acc[0] += v.x;
                acc[1] += v.y;
                acc[2] += v.z;
                acc[3] += v.w;
            }
            if (d.rec < 0) {
                const int j = (d.row0 + r) / G, h = d.kvh * G + (d.row0 + r) % G;
                float val[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) val[k] = L == 0.f ? 0.f : acc[k] / L;  // (a NaN stays one)
                store4_from_f32(a.out, a.out_dtype, (((size_t)d.b * a.rows + j) * a.num_q_heads + h) * HD + dim, val);
            } else {
                const size_t p = (size_t)d.rec * (16 * NT) + r;
                store_agent2(a.ws_acc + p * HD + dim, acc[0], acc[1]);
                store_agent2(a.ws_acc + p * HD + dim + 2, acc[2], acc[3]);
                if (dim == 0) store_agent2(a.ws_ml + p * 2, mx > -1e29f ? mx * kLn2 : -1e30f, L);
            }
        }
        __syncthreads();
    }
}

// PLANNED: workgroup p runs the plan's piece p, and the last piece of a split item merges it. Else
// workgroup (sequence, head) runs the whole item: calls too narrow to cut, and batches that the
// plan does not rank.
template <int NT, int HD, bool PREC, int TOK, bool PLANNED>
__global__ void __launch_bounds__(256, NT == 1 && TOK == 32 ? 4 : 2) attn_int4_kernel(AttnArgs a, KVView kv) {
    const int heads = kv.Hkv * a.row_groups;
    if constexpr (PLANNED) {
        const int p = blockIdx.x;
        const int4 e = ((const int4*)lpt_table(a.plan))[2 * p], f = ((const int4*)lpt_table(a.plan))[2 * p + 1];
        if (e.x < 0) return;  // past the last piece
        const int h = e.y & 0xffff, np = e.y >> 16, row0 = h / kv.Hkv * (16 * NT);
        const PieceDesc d{e.x, h % kv.Hkv, e.z, e.w, -1, np > 1 ? f.z + f.w * heads : -1, row0, f.x, f.y};
        int4_piece<NT, HD, PREC, TOK>(a, kv, d);
        if (np > 1 && a.num_q_heads / kv.Hkv * d.nrows > row0) lpt_merge_if_last<HD>(a, kv.Hkv, heads, d, h, np, f.z, 16 * NT);
    } else {
        const int h = blockIdx.x % heads, b = blockIdx.x / heads;
        const int ctx = seq_keys(a, b, kBS), nrows = seq_rows(a, b);
        int4_piece<NT, HD, PREC, TOK>(a, kv, PieceDesc{b, h % kv.Hkv, 0, ctx, -1, -1, h / kv.Hkv * (16 * NT), ctx, nrows});
    }
}

template <int NT, int HD, bool PREC, int TOK>
void launch_one(const AttnArgs& a, const KVView& kv, hipStream_t s) {
    if (a.sched == ATTN_SCHED_LPT)
        attn_int4_kernel<NT, HD, PREC, TOK, true><<<lpt_pieces(a.sk_grid, a.num_seqs, kv.Hkv * a.row_groups), 256, 0, s>>>(a, kv);
    else
        attn_int4_kernel<NT, HD, PREC, TOK, false><<<a.num_seqs * kv.Hkv * a.row_groups, 256, 0, s>>>(a, kv);
}

template <int NT, int HD, int TOK>
void launch_prec(const AttnArgs& a, const KVView& kv, hipStream_t s) {
    if (a.q_dtype == GG_DTYPE_F32 || a.out_dtype == GG_DTYPE_F32) launch_one<NT, HD, true, TOK>(a, kv, s);
    else launch_one<NT, HD, false, TOK>(a, kv, s);
}

// (int4_chunk_tokens: 64 or 32 at one row tile, 64 at two, 32 at three and four.)
template <int HD>
void launch_tiles(const AttnArgs& a, const KVView& kv, int nt, int tok, hipStream_t s) {
    if (nt == 1 && tok == 64) launch_prec<1, HD, 64>(a, kv, s);
    else if (nt == 1) launch_prec<1, HD, 32>(a, kv, s);
    else if (nt == 2) launch_prec<2, HD, 64>(a, kv, s);
    else if (nt == 3) launch_prec<3, HD, 32>(a, kv, s);
    else if constexpr (HD == 64) launch_prec<4, HD, 32>(a, kv, s);
}

}  // namespace

gg_status_t launch_attn_int4(const AttnArgs& a, const KVView& kv, const AttnShape& sh, int tok, hipStream_t s) {
    if (kv.D == 128) launch_tiles<128>(a, kv, sh.nt, tok, s);
    else launch_tiles<64>(a, kv, sh.nt, tok, s);
    return check_hip(hipGetLastError(), "verify_attention launch");
}

}  // namespace gg
