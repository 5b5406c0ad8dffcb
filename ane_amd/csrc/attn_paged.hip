// attn_paged.hip — attention of one new token over a paged cache of keys and values.
//   p_t = exp(scale q.k_t - lse) for 0 <= t <= pos,  o = sum_t p_t v_t,  lse = log sum_t exp(scale q.k_t)
//
// Every key and value is read once for the query heads that share it, and little is computed with it: the time is that of reading the cache.
// So a wave takes tiles of 32 positions (fp32: 16), 16 KB of keys and values at 128 channels, straight into registers, the next tile under way
// while one is used, with nothing shared between waves and no barrier on the way: eight waves to a compute unit keep 128 KB in flight.
//
// Both products run on the matrix cores, with up to 16 query heads of a KV head for their columns (a group of two leaves 14 of them empty, and the
// products still take a tenth of the time that the reading does):
//   scores[position][head] = K q:  a lane's operand is 16 bytes of a row of the cache, position lane % 16, as it lies in memory;
//   o[channel][head] += V' p:      p is taken from the registers that the scores are in: register r of lane l is position 4 (l / 16) + r, so the
//                                  lane reads the values of just these positions.  In bfloat16 an operand is eight positions of a
//                                  channel: the lane holds eight rows of 8 (4) channels and exchanges halves of words between them.
// The running maximum is brought up to date only when a score passes it, which is rare after the first tiles, so lanes hardly ever talk.
//
// Measured, pages of 16: 64 sequences of up to 4096 positions, 16 heads on 8 KV heads of 128, bfloat16, 91.7 us for 421 MB, 4.6 TB/s; one of 131071
// (pages of 64) 107 us, 5.0 TB/s, where a copy of 1 GiB reaches 5.1: bound by HBM.  64 of up to 200 14.4 us, one of 256 8.7; 12 heads of 64, fp32,
// 8.3: bound by one load after the other (positions, a page, a tile, the parts of a result).  (Workgroups of 2 waves instead of 4 took 125 us for the
// long one when that took 108, of 8 102, but one of 256 9.3 instead of 8.7.)
//
// Two waves to a SIMD, with half of its registers each.  In fp32 a wave takes 136 to 247 vector registers, by the head's size, and 45 to 53 scalar
// ones are kept in lanes of vector registers.  In bfloat16 it is 248 to 256 for any size, 105 to 123 and 56 to 448 bytes of private memory: the rare
// second pass (share_out_again) is a call, and what is alive across it is kept as its convention has it.
#include "deal.h"
#include "kv_cache.h"
#include "mma.h"

#include <math.h>

namespace {

constexpr float LOG2E = 1.44269502162933349609375f, LN2 = 0.693147182464599609375f;
constexpr float FAR = 16777216.f;           // 2^24
constexpr int HEADS = 16;                   // query heads of one product
constexpr int WAVES = 4;
constexpr int MAX_GROUPS = 1024;            // workgroups of a launch
// In tiles, of which a workgroup's waves have one each at a time: what beginning another unit takes, what a workgroup should have at least, and what is
// not cut off a unit.  us, pages of 16, bfloat16, 16 heads on 8 KV heads of 128, unless said otherwise:
//                                              as it is   GRAIN 16 / 32    BEGIN 1   SHORT 1
//   one sequence of 256, 12 heads of 64, fp32      8.3       8.3 / 12.9       8.4       9.2
//   one of 256                                     8.7       8.8 / 13.9       8.8       8.7
//   one of 2048                                   13.6      15.6 / 19.6      13.4      11.6
//   64 of up to 200                               14.5      17.2 / 19.7      19.3      17.5
//   64 of up to 4096                              91.7      91.7 / 91.9      91.6      90.5
//   9 of up to 7892, 40 heads on two, pages of 64 23.3      27.8 / 35.6      23.4      25.7
//   16 of up to 8000, 40 heads on two, the same   31.0      31.4 / 38.4      30.7      36.3
constexpr int BEGIN = 8, GRAIN = 8, SHORT = 9;
// Joining costs by the heads.  us, GRAIN / twice that for all: 64 heads on one KV head, 16 of up to 4000, 27.8 / 23.0, 8 of up to 1000, 16 heads on 8,
// 13.6 / 15.6, but 3 of up to 449, 40 heads on two, fp32, 15.4 / 17.0.
constexpr __host__ __device__ int grain(int heads) { return heads >= 8 ? 2 * GRAIN : GRAIN; }
// Few units of many tiles should not be cut into as many pieces as there are workgroups: a piece takes as long as it has tiles, the join as long as
// there are pieces and heads, and both together least at pieces of about sqrt(tiles heads) / 3.  us, without / with that, one sequence of 65536
// positions: 6 heads of 96 on one, fp32, 94.6 / 35.0, 40 of 128 on two, bfloat16, 66.9 / 38.8, 64 on one 65.4 / 41.7; of 131071, 8 heads on one
// 61.9 / 39.1.  Not where it leaves more than one workgroup to a compute unit but fewer than two: those take as long as two each (6 of up to 46491, 40
// heads on two, 62 instead of 51).
constexpr float PIECE = 1.f / 3;
// Slots whose values a thread has on their way at once.  us, 6 / 8 / 12: one sequence of 65536 positions, 6 heads on one KV head, fp32, 38.9 / 36.8 /
// 35.0, 40 on two 42.5 / 40.8 / 38.8, 6 of up to 46491 53.8 / 52.8 / 51.7, 64 heads on one, 16 of up to 4000, 23.9 / 23.2 / 23.2, one of 256 8.7 / 8.7 / 8.7.
constexpr int JOIN = 12;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct PagedArgs {
    mi355_kv_cache c;
    const int *seq, *pos;
    int heads, S, col0, cols;       // columns col0 .. col0 + cols - 1
    int group, positions;           // query heads of a KV head; positions of a row of the table
    int part0, parts, units;        // which parts of the groups this launch has; compute units, 0 where units are not long enough for PIECE to matter
    float scale2;
    float *slots;                   // partial results: two for each workgroup
    unsigned *arrived;
};

// ---- the parts of a tile that depend on the type ----

// 16 bytes at `at` of the lane and `row` of the wave
template <typename V>
__device__ __forceinline__ V load16(__amdgpu_buffer_rsrc_t from, unsigned at, unsigned row) {
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(from, (int)at, (int)row, 0));
}

template <typename T, int HDB> struct Tile;

template <int HDB> struct Tile<bf16_t, HDB> {
    static constexpr int PIECES = 2, POSITIONS = 32;            // pieces of 16 positions, each in one page
    static constexpr int VC = HDB > 2 ? 8 : 4, ACC = VC;        // channels of V to a lane; products of 16 channels each
    typedef unsigned Vec __attribute__((ext_vector_type(VC / 2), aligned(VC * 2)));
    typedef bf16x8 Q;
    static constexpr int QS = HDB;
    v4u k[PIECES][HDB];
    Vec v[8];
    static __device__ __forceinline__ int channel(int acc, int r, int g) { return VC * (4 * g + r) + acc; }
    static __device__ __forceinline__ Q query(const float *row, int s) {        // LDS: fp32 values of a head
        const float *p = row + 32 * s + 8 * ((threadIdx.x & 63) >> 4);
        const v4u w = {f2_to_bf2(p[0], p[1]), f2_to_bf2(p[2], p[3]), f2_to_bf2(p[4], p[5]), f2_to_bf2(p[6], p[7])};
        return __builtin_bit_cast(Q, w);
    }
    // Bytes from the first of a piece's 16 rows to what the lane reads of them; channels behind the last are read as zero.
    struct Offsets { unsigned k, k_last, v, row; };
    static __device__ __forceinline__ Offsets offsets(int hd) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, tail = 32 * (HDB - 1) + 8 * g;
        return {(unsigned)(i * hd + 8 * g) * 2, tail < hd ? (unsigned)(i * hd + tail) * 2 : OUTSIDE,
                VC * i < hd ? (unsigned)(4 * g * hd + VC * i) * 2 : OUTSIDE, (unsigned)hd * 2};
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, int piece, const Offsets &o) {
#pragma unroll
        for (int s = 0; s < HDB; s++) k[piece][s] = load16<v4u>(kr, s < HDB - 1 ? o.k + 64 * s : o.k_last, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if constexpr (VC == 8) v[4 * piece + r] = load16<Vec>(vr, o.v, r * o.row);
            else v[4 * piece + r] = __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b64(vr, (int)o.v, (int)(r * o.row), 0));
        }
    }
    __device__ __forceinline__ v4f scores(const Q (&q)[QS], int piece) const {
        v4f s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < HDB; j++) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[piece][j]), q[j], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void hide(int piece, int r) { v[4 * piece + r] = Vec(0u); }
    // acc += V' p.  A weight is a pair of bfloat16 values, its upper half and what that leaves of it: off by 2^-15 of it, where one value
    // alone is off by as much as the rounding of the result (2^-8).  ODD: infinities and NaNs among the values count as zero.
    // (A third value would leave nothing out.  Relative error of o, 64 sequences of up to 4096 positions: 0.00166210 with two, 0.00166209 with three or
    // fp32 weights, all of it the rounding of o, of which 0.36 % and 0.05 % come out as the neighbouring value.  us, two / three: that call 91.4 / 91.7,
    // one of 65536, 40 heads on two, 39.2 / 44.7, 64 on one 41.8 / 46.2, 6 of up to 46491, 40 on two, 51.7 / 55.0.)
    template <bool ODD>
    __device__ __forceinline__ void weigh(v4f (&acc)[ACC], const v4f (&p)[PIECES]) const {
        v4u hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = p[i >> 1][2 * (i & 1)], y = p[i >> 1][2 * (i & 1) + 1];
            const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
            hi[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            float ra = x - __uint_as_float(a & 0xffff0000u), rb = y - __uint_as_float(b & 0xffff0000u);
            lo[i] = f2_to_bf2(ra, rb);
        }
#pragma unroll
        for (int c = 0; c < VC; c++) {
            v4u w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_perm(v[2 * i + 1][c >> 1], v[2 * i][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
            if (ODD) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
                    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
                }
            }
            const bf16x8 a = __builtin_bit_cast(bf16x8, w);
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, lo), acc[c], 0, 0, 0);
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, hi), acc[c], 0, 0, 0);
        }
    }
};

template <int HDB> struct Tile<float, HDB> {
    static constexpr int PIECES = 1, POSITIONS = 16;
    static constexpr int WIDE = HDB > 2 ? 2 : 1, ACC = 4 * WIDE;        // 16 lanes read 64 channels of a row at a time
    typedef v4f Q;
    static constexpr int QS = 2 * HDB;
    v4f k[2 * HDB], v[4][WIDE];
    static __device__ __forceinline__ int channel(int acc, int r, int g) { return 64 * (acc >> 2) + 4 * (4 * g + r) + (acc & 3); }
    static __device__ __forceinline__ Q query(const float *row, int s) {
        return *reinterpret_cast<const v4f *>(row + 16 * s + 4 * ((threadIdx.x & 63) >> 4));
    }
    struct Offsets { unsigned k, k_tail[2], v, v_last, row; };
    static __device__ __forceinline__ Offsets offsets(int hd) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, tail = 32 * (HDB - 1) + 4 * g, last = 64 * (WIDE - 1) + 4 * i;
        return {(unsigned)(i * hd + 4 * g) * 4,
                {tail < hd ? (unsigned)(i * hd + tail) * 4 : OUTSIDE, tail + 16 < hd ? (unsigned)(i * hd + tail + 16) * 4 : OUTSIDE},
                (unsigned)(4 * g * hd + 4 * i) * 4, last < hd ? (unsigned)(4 * g * hd + last) * 4 : OUTSIDE, (unsigned)hd * 4};
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, int, const Offsets &o) {
#pragma unroll
        for (int s = 0; s < 2 * HDB; s++)
            k[s] = load16<v4f>(kr, s < 2 * HDB - 2 ? o.k + 64 * s : o.k_tail[s & 1], 0);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int w = 0; w < WIDE; w++) v[r][w] = load16<v4f>(vr, w < WIDE - 1 ? o.v : o.v_last, r * o.row);
    }
    __device__ __forceinline__ v4f scores(const Q (&q)[QS], int) const {
        v4f s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2 * HDB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][e], q[j][e], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void hide(int, int r) {
#pragma unroll
        for (int w = 0; w < WIDE; w++) v[r][w] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    template <bool ODD>
    __device__ __forceinline__ void weigh(v4f (&acc)[ACC], const v4f (&p)[PIECES]) const {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int w = 0; w < WIDE; w++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][w][e], p[0][r], acc[4 * w + e], 0, 0, 0);
    }
};

// ---- a walk over tiles of one sequence and KV head ----

// Where a wave's pieces lie: lane j has the page and the place in it of the j-th of 64 of them (-1 behind the sequence's end).  A wave
// looks 64 up at once, long before it needs them: waiting for one number of the table would wait for all loads of keys and values before it.
struct Pieces {
    int id, slot;
    // PIECES of tile first, of tile first + WAVES, ...
    template <int PIECES>
    __device__ __forceinline__ void look_up(const int *table, int page, int len, int first) {
        const int j = threadIdx.x & 63, per_page = page >> 4;
        const int piece = (first + j / PIECES * WAVES) * PIECES + j % PIECES;
        const unsigned at = (unsigned)piece / (unsigned)per_page;
        slot = piece - (int)at * per_page;
        id = -1;
        if (piece < (len + 15) >> 4) id = table[at];        // (looked at when it is needed: see places())
    }
};

template <typename T, int HDB>
struct Walk {
    typedef Tile<T, HDB> Tl;
    v4f acc[Tl::ACC];
    float m, l;
    bool seen;

    struct Place { int id[Tl::PIECES], slot[Tl::PIECES]; };
    static constexpr int BATCH = 64 / Tl::PIECES;           // tiles whose pages are looked up at once
    static __device__ __forceinline__ Place places(const Pieces &in, int i, int n_pages) {
        Place p;
#pragma unroll
        for (int j = 0; j < Tl::PIECES; j++) {
            const int id = __builtin_amdgcn_readlane(in.id, (i % BATCH) * Tl::PIECES + j);
            p.id[j] = paged_id_ok(id, n_pages) ? id : -1;
            p.slot[j] = __builtin_amdgcn_readlane(in.slot, (i % BATCH) * Tl::PIECES + j);
        }
        return p;
    }

    // tile: its number; ids: its pages
    template <bool ODD>
    __device__ __forceinline__ void use(Tl &t, const Place &p, const typename Tl::Q (&q)[Tl::QS], int tile, int len, int hd, float scale2, const T *v,
                                        size_t page_stride) {
        const int g = (threadIdx.x & 63) >> 4;
        bool whole = (tile + 1) * Tl::POSITIONS <= len;
#pragma unroll
        for (int i = 0; i < Tl::PIECES; i++) {
            const bool ok = p.id[i] >= 0;
            whole &= ok;
            seen |= ok;
        }
        v4f s[Tl::PIECES];
#pragma unroll
        for (int i = 0; i < Tl::PIECES; i++) s[i] = t.scores(q, i);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < Tl::PIECES; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (!(p.id[i] >= 0 && tile * Tl::POSITIONS + 16 * i + 4 * g + r < len)) {
                        s[i][r] = -INFINITY;
                        t.hide(i, r);
                    }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < Tl::PIECES; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[i][r]);
        mx *= scale2;
        if (__any(mx > m)) {        // the running maximum moves: what is there is brought to the new one
            mx = fmaxf(mx, lane_xor<16>(mx));
            mx = fmaxf(mx, lane_xor<32>(mx));
            const float to = fmaxf(m, mx), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int a = 0; a < Tl::ACC; a++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[a][r] *= f;
            m = to;
        }
        const float base = m == -INFINITY ? 0.f : m;
        // m is rounded and the fused product is not: their difference, up to 2^-24 m, is in every weight and in their sum alike, until it is
        // beyond what an exponential holds.  From FAR on products are rounded as m is, and the largest is exactly 0 off.
        float by = scale2;
        if (__any(fabsf(base) > FAR)) {
            const bool far = fabsf(base) > FAR;
#pragma unroll
            for (int i = 0; i < Tl::PIECES; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[i][r] = far ? s[i][r] * scale2 : s[i][r];
            by = far ? 1.f : scale2;
        }
#pragma unroll
        for (int i = 0; i < Tl::PIECES; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], by, -base));
                l += s[i][r];
            }
        t.template weigh<ODD>(acc, s);
        if constexpr (ODD) {
            // the infinities and NaNs that were left out of the product, one position after the other
#pragma unroll 1
            for (int x = 0; x < Tl::POSITIONS; x++) {
                const int i = x >> 4, r = x & 3;
                const float w0 = i ? s[Tl::PIECES - 1][0] : s[0][0], w1 = i ? s[Tl::PIECES - 1][1] : s[0][1], w2 = i ? s[Tl::PIECES - 1][2] : s[0][2],
                            w3 = i ? s[Tl::PIECES - 1][3] : s[0][3];
                const float w = __shfl(r == 0 ? w0 : r == 1 ? w1 : r == 2 ? w2 : w3, (threadIdx.x & 15) + ((x >> 2 & 3) << 4), 64);
                const int id = i ? p.id[Tl::PIECES - 1] : p.id[0], slot = i ? p.slot[Tl::PIECES - 1] : p.slot[0];
                if (id < 0 || tile * Tl::POSITIONS + x >= len) continue;
                const T *row = v + id * page_stride + (size_t)(slot * 16 + (x & 15)) * hd;
#pragma unroll
                for (int a = 0; a < Tl::ACC; a++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int ch = Tl::channel(a, e, g);
                        const float y = ch < hd ? load_one(row + ch) : 0.f;
                        if (!is_finite(y)) acc[a][e] += w * y;
                    }
            }
        }
    }

    // Tiles first, first + WAVES, ... below last.  k, v: the KV head's rows of page 0.
    // now: the pages of the first 64 pieces.
    template <bool ODD>
    __device__ __forceinline__ void run(const typename Tl::Q (&q)[Tl::QS], Pieces now, const T *k, const T *v, size_t page_stride, const int *table,
                                        int page, int n_pages, int hd, int first, int last, int len, float scale2) {
        m = -INFINITY;
        l = 0.f;
        seen = false;
#pragma unroll
        for (int a = 0; a < Tl::ACC; a++) acc[a] = v4f{0.f, 0.f, 0.f, 0.f};
        if (first >= last) return;
        const typename Tl::Offsets offsets = Tl::offsets(hd);
        auto load = [&](Tl &t, const Place &p) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < Tl::PIECES; i++) {
                const size_t o = (size_t)max(p.id[i], 0) * page_stride + (size_t)(p.slot[i] * 16) * hd;
                const int bytes = p.id[i] < 0 ? 0 : 16 * hd * (int)sizeof(T);      // a piece of no page is read as zeros
                t.load(__builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(k + o), 0, bytes, 0x00027000),
                       __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(v + o), 0, bytes, 0x00027000), i, offsets);
            }
        };
        Pieces then;
        Tl a, b;
        Place pa = places(now, 0, n_pages), pb;
        load(a, pa);
        then.look_up<Tl::PIECES>(table, page, len, first + BATCH * WAVES);
        // tile i is used while tile i + 1 is under way
        auto ahead = [&](Tl &t, Place &p, int i) __attribute__((always_inline)) {
            if (i % BATCH == 0) {
                now = then;
                then.look_up<Tl::PIECES>(table, page, len, first + (i + BATCH) * WAVES);
            }
            p = places(now, i, n_pages);
            // (behind the last one nothing; but a load behind a condition would have the compiler wait for all of them)
            if (first + i * WAVES >= last) {
#pragma unroll
                for (int j = 0; j < Tl::PIECES; j++) p.id[j] = -1;
            }
            load(t, p);
        };
        for (int i = 0;; i += 2) {
            ahead(b, pb, i + 1);
            use<ODD>(a, pa, q, first + i * WAVES, len, hd, scale2, v, page_stride);
            if (first + (i + 1) * WAVES >= last) break;
            ahead(a, pa, i + 2);
            use<ODD>(b, pb, q, first + (i + 1) * WAVES, len, hd, scale2, v, page_stride);
            if (first + (i + 2) * WAVES >= last) break;
        }
        l += lane_xor<16>(l);
        l += lane_xor<32>(l);
    }
};

// What the waves of a workgroup leave one another of the unit at hand.
template <int HDB>
struct Shared {
    static constexpr int ROW = HDB * 32 + 4;
    float q[HEADS * ROW], o[WAVES * HEADS * ROW];       // the queries as fp32 values; each wave's o
    float m[WAVES * HEADS], l[WAVES * HEADS];
    int seen[WAVES];
    __device__ __forceinline__ float sum_at(int h, int ch) const {
        const float *p = o + h * ROW + ch;
        return ((p[0] + p[HEADS * ROW]) + p[2 * HEADS * ROW]) + p[3 * HEADS * ROW];
    }
    __device__ __forceinline__ void stats(int h, float &top, float &sum) const {
        top = fmaxf(fmaxf(m[h], m[HEADS + h]), fmaxf(m[2 * HEADS + h], m[3 * HEADS + h]));
        const float base = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; i++) sum += l[i * HEADS + h] * __builtin_amdgcn_exp2f(m[i * HEADS + h] - base);
    }
};
template <int HDB> using shared_ptr = __attribute__((address_space(3))) Shared<HDB> *;

// Tiles t0 .. t1 - 1 of a sequence and KV head: the waves' shares, brought to the largest of their maxima, are in LDS at the end.
template <typename T, int HDB, bool ODD>
__device__ __forceinline__ void share_out(shared_ptr<HDB> lds_, Pieces now, const T *k, const T *v, size_t page_stride, const int *table, int page,
                                          int n_pages, int hd, int heads, int t0, int t1, int len, float scale2) {
    typedef Tile<T, HDB> Tl;
    Shared<HDB> &lds = *(Shared<HDB> *)lds_;
    constexpr int ROW = Shared<HDB>::ROW;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), g = lane >> 4, head = lane & 15;
    typename Tl::Q q[Tl::QS];
#pragma unroll
    for (int i = 0; i < Tl::QS; i++) q[i] = Tl::query(lds.q + head * ROW, i);
    Walk<T, HDB> walk;
    walk.template run<ODD>(q, now, k, v, page_stride, table, page, n_pages, hd, t0 + wave, t1, len, scale2);
    if (g == 0) {
        lds.m[wave * HEADS + head] = walk.m;
        lds.l[wave * HEADS + head] = walk.l;
    }
    if (lane == 0) lds.seen[wave] = walk.seen;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < WAVES; i++) top = fmaxf(top, lds.m[i * HEADS + head]);
    const float f = __builtin_amdgcn_exp2f(walk.m - (top == -INFINITY ? 0.f : top));
    if (head < heads) {
#pragma unroll
        for (int x = 0; x < Tl::ACC; x += 4)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int ch = Tl::channel(x, r, g);            // and the three behind it
                if (ch < HDB * 32)
                    *reinterpret_cast<v4f *>(lds.o + (wave * HEADS + head) * ROW + ch) =
                        v4f{walk.acc[x][r] * f, walk.acc[x + 1][r] * f, walk.acc[x + 2][r] * f, walk.acc[x + 3][r] * f};
            }
    }
    __syncthreads();
}
// The same with infinities and NaNs among the values taken one by one; a function of its own, for its registers not to be the kernel's.
template <typename T, int HDB>
__device__ __attribute__((noinline)) void share_out_again(shared_ptr<HDB> lds, const T *k, const T *v, size_t page_stride, const int *table, int page,
                                                          int n_pages, int hd, int heads, int t0, int t1, int len, float scale2) {
    Pieces now;
    now.look_up<Tile<T, HDB>::PIECES>(table, page, len, t0 + uniform((int)threadIdx.x >> 6));
    share_out<T, HDB, true>(lds, now, k, v, page_stride, table, page, n_pages, hd, heads, t0, t1, len, scale2);
}

// Two values of a slot.  Slots pass from one workgroup to another inside a launch without fences, which would write back and invalidate whole L2s:
// such stores go through to memory and such loads do not stop at the L2, and the count of those that have arrived goes up when the stores of a
// workgroup have ended.
__device__ __forceinline__ void slot_put(float *p, float x, float y) {
    const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store((unsigned long long *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ v2f slot_get(const float *p) {
    const unsigned long long v = __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return v2f{__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32))};
}

// A unit is the tiles of a column and KV head.  Those of all columns, one after the other, are dealt out evenly, a unit
// counted as its tiles and BEGIN more for what it takes to begin one: workgroup w of W has T / W of that line, whatever sequences they belong to.
// (Lengths are in device memory: the host cannot deal them out, and a batch's longest sequence would otherwise decide when it ends.)  A border that
// would cut off fewer than SHORT tiles is moved to the unit's end or beginning.  A unit with borders inside is split: each of its workgroups
// leaves its maxima, sums and unnormalised o in a slot, and the last one to arrive joins them in their order.  A workgroup has two such units at
// most, the one that it begins with and the one that it ends with, and looks after both when it is done with its tiles.
// More than 16 query heads to a KV head go in parts, each with workgroups, slots and counts of its own.  Those with the same tiles lie 8 apart in the grid:
// they begin together on one XCD, and what the first one reads the others find in its L2.  (40 heads on two KV heads, 6 sequences of up to 46491 positions
// 64.5 -> 54.2 us, 16 of up to 8000 37.3 -> 32.4, where parts followed one another on one line.)
template <typename T, int HDB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void attn_paged_kernel(T *__restrict__ o, float *__restrict__ lse, const T *__restrict__ q, PagedArgs a) {
    typedef Tile<T, HDB> Tl;
    constexpr int ROW = Shared<HDB>::ROW;
    __shared__ __attribute__((aligned(16))) Shared<HDB> lds;
    __shared__ int sums[WAVES], ticket[2];
    __shared__ float tops[WAVES];
    __shared__ struct { int col, unit, tile, start, len; } ends[2];
    const int tid = threadIdx.x, hd = a.c.hd, page = a.c.page;
    const int all_parts = (a.group + HEADS - 1) / HEADS, part_heads = (a.group + all_parts - 1) / all_parts;
    const int units = a.c.kv_heads;         // of a column
    const int turn = blockIdx.x / (8 * a.parts), rest = blockIdx.x - turn * 8 * a.parts, part = a.part0 + (rest >> 3), w = turn * 8 + (rest & 7);
    const int heads = min(a.group - part * part_heads, part_heads), most = gridDim.x / a.parts;
    auto length = [&](int col) __attribute__((always_inline)) {
        const int p = a.pos[col], seq = a.seq ? a.seq[col] : col;
        return seq < 0 || seq >= a.c.n_seqs || p < 0 || p >= a.positions ? 0 : p + 1;
    };
    auto tiles_of = [&](int col) __attribute__((always_inline)) { return (length(col) + Tl::POSITIONS - 1) / Tl::POSITIONS; };
    auto weight_of = [&](int col) __attribute__((always_inline)) {
        const int n = tiles_of(col);
        return n ? (n + BEGIN) * units : 0;
    };

    // where this workgroup's tiles begin and end
    const int each = (a.cols + 255) / 256, c0 = min(tid * each, a.cols), c1 = min(c0 + each, a.cols);
    // (Up to 256 columns a thread has one, whose length it keeps: looked up again it is waited for three times more, and calls of 8 to 65 us take
    // 0.4 us longer.)
    const int len0 = c0 < c1 ? length(a.col0 + c0) : 0, n0 = (len0 + Tl::POSITIONS - 1) / Tl::POSITIONS;
    int mine = n0 ? (n0 + BEGIN) * units : 0;
    float longest = n0;
    for (int c = c0 + 1; c < c1; c++) {
        const int n = tiles_of(a.col0 + c);
        mine += n ? (n + BEGIN) * units : 0;
        longest = fmaxf(longest, n);
    }
    if (a.units) longest = wave_max(longest);
    for (int i = tid; i < HEADS * ROW; i += 256) lds.q[i] = 0.f;           // (heads that there are not)
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(upto, d, 64);
        if ((tid & 63) >= d) upto += x;
    }
    if ((tid & 63) == 63) {
        sums[tid >> 6] = upto;
        tops[tid >> 6] = longest;
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        if (i < tid >> 6) upto += sums[i];
        total += sums[i];
        longest = fmaxf(longest, tops[i]);
    }
    total = uniform(total);
    int groups = deal_groups(total, most, grain(part_heads));
    // (a multiple of the units: a workgroup that ends one and begins another is often the last of both, and joins one after the other)
    if (a.units) groups = deal_fewer(groups, total, max(1, uniform((int)(sqrtf(longest * part_heads) * PIECE))), units, a.units / a.parts);
    if (w >= groups) return;
    const Deal deal = deal_out(total, groups);
    // The column, unit and tile of a border: the thread whose columns have it walks over them.
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int x = deal.border(w + i);
        if (x >= upto - mine && x < upto) {
            int b = upto - mine, c = a.col0 + c0, len = len0;
            if (each > 1) {
                while (x >= b + weight_of(c)) b += weight_of(c++);
                len = length(c);
            }
            const int n = (len + Tl::POSITIONS - 1) / Tl::POSITIONS;
            const DealPlace at = deal_place(x - b, n, BEGIN, SHORT);
            ends[i].col = c;
            ends[i].unit = at.unit;
            ends[i].tile = at.tile;
            ends[i].start = b;
            ends[i].len = len;
        }
        if (x == total && tid == 0) ends[i] = {a.col0 + a.cols, 0, 0, total, 0};
    }
    __syncthreads();
    int col = uniform(ends[0].col), unit = uniform(ends[0].unit), tile = uniform(ends[0].tile);
    int start = uniform(ends[0].start), len = uniform(ends[0].len);         // of the column
    const int end_col = uniform(ends[1].col), end_unit = uniform(ends[1].unit), end_tile = uniform(ends[1].tile);
    const size_t page_stride = (size_t)a.c.kv_heads * page * hd, slot_size = (size_t)HEADS * (HDB * 32 + 2);
    const int row = hd + 2;             // of a slot: a head's maximum, its sum (-1: no position seen), its channels
    float *const slots = a.slots + (size_t)(part - a.part0) * most * 2 * slot_size;
    unsigned *const arrived = a.arrived + (part - a.part0) * most;
    // the unit that began before, the one that ends behind
    struct Split { int col, kvh, first, last; } split[2] = {{-1, 0, 0, 0}, {-1, 0, 0, 0}};
    auto out_of = [&](int col, int head0, size_t channels) __attribute__((always_inline)) {
        const int b = col / a.S, s = col - b * a.S;
        return ((size_t)b * a.heads + head0) * channels * a.S + s;
    };

    while (col < end_col || (col == end_col && (unit < end_unit || (unit == end_unit && tile < end_tile)))) {
        const int n = (len + Tl::POSITIONS - 1) / Tl::POSITIONS;
        if (n == 0 || unit == units) {
            if (n) start += (n + BEGIN) * units;
            col++;
            unit = tile = 0;
            if (col < a.col0 + a.cols) len = uniform(length(col));
            continue;
        }
        const int kvh = unit, t0 = tile, t1 = col == end_col && unit == end_unit ? end_tile : n;
        const int head0 = kvh * a.group + part * part_heads, seq = uniform(a.seq ? a.seq[col] : col);
        const T *k = (const T *)a.c.k + (size_t)kvh * page * hd, *v = (const T *)a.c.v + (size_t)kvh * page * hd;
        const int *table = a.c.pages + (size_t)seq * a.c.max_pages;
        Pieces now;
        now.look_up<Tl::PIECES>(table, page, len, t0 + uniform(tid >> 6));
        const T *qp = q + out_of(col, head0, hd);
        // the queries, as fp32 values
        for (int i = tid; i < heads * hd; i += 256) {
            const int h = i / hd;
            lds.q[h * ROW + i - h * hd] = load_one(qp + (size_t)i * a.S);
        }
        __syncthreads();
        share_out<T, HDB, false>((shared_ptr<HDB>)&lds, now, k, v, page_stride, table, page, a.c.n_pages, hd, heads, t0, t1, len, a.scale2);
        if constexpr (sizeof(T) == 2) {
            // An infinity times the half of a weight that is zero is NaN: such sums are formed again.
            bool odd = false;
            for (int i = tid; i < heads * hd; i += 256) {
                const int h = i / hd;
                const float x = lds.sum_at(h, i - h * hd);
                odd |= x != x;
            }
            if (__syncthreads_or(odd))
                share_out_again<T, HDB>((shared_ptr<HDB>)&lds, k, v, page_stride, table, page, a.c.n_pages, hd, heads, t0, t1, len, a.scale2);
        }
        const bool any = lds.seen[0] | lds.seen[1] | lds.seen[2] | lds.seen[3];
        if (t0 == 0 && t1 == n) {
            T *op = o + out_of(col, head0, hd);
            if (any)
                for (int i = tid; i < heads * hd; i += 256) {
                    const int h = i / hd;
                    float top, sum;
                    lds.stats(h, top, sum);
                    store_one(op + (size_t)i * a.S, lds.sum_at(h, i - h * hd) / sum);
                    if (lse && i == h * hd) lse[out_of(col, head0 + h, 1)] = (top + __builtin_amdgcn_logf(sum)) * LN2;
                }
        } else {
            float *slot = slots + ((size_t)w * 2 + (t0 == 0)) * slot_size;
            for (int i = 2 * tid; i < heads * row; i += 512) {
                const int h = i / row, x = i - h * row;
                float v0, v1;
                if (x == 0) {
                    lds.stats(h, v0, v1);
                    v1 = any ? v1 : -1.f;
                } else v0 = lds.sum_at(h, x - 2), v1 = lds.sum_at(h, x - 1);
                slot_put(slot + i, v0, v1);
            }
            const DealShared shared = deal_shared(deal, start + unit * (n + BEGIN), n, BEGIN, SHORT);
            split[t0 == 0] = {col, kvh, shared.first, shared.last};
        }
        __syncthreads();
        unit++;
        tile = 0;
    }

    if (split[0].col < 0 && split[1].col < 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // this wave's parts of the slots are in memory,
    __syncthreads();                                        // everybody's are
    if (tid < 2 && (tid ? split[1].col : split[0].col) >= 0)
        ticket[tid] = (int)__hip_atomic_fetch_add(arrived + (tid ? split[1].first : split[0].first), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        const Split u = i ? split[1] : split[0];
        if (u.col < 0 || ticket[i] != u.last - u.first) continue;
        // The last to arrive: everybody's slots are in memory.
        if (tid == 0) __hip_atomic_store(arrived + u.first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int head0 = u.kvh * a.group + part * part_heads, count = u.last - u.first + 1;
        T *op = o + out_of(u.col, head0, hd);
        // four channels to a thread (two: 5 to 7 % longer with ten heads and more), and the slots in turns where there are threads to spare
        const int quads = heads * hd / 4, turns = min(max(1, 256 / quads), (count + 1) / 2);
        for (int x0 = 0; x0 < quads * turns; x0 += 256) {
            const int x = x0 + tid, turn = x / quads, quad = x - turn * quads, h = 4 * quad / hd, ch = 4 * quad - h * hd;
            const bool in = x < quads * turns;
            const float *mine = slots + ((size_t)u.first * 2) * slot_size + h * row;
            float top = -INFINITY, sum = -1.f;
            v4f v = {0.f, 0.f, 0.f, 0.f};
            for (int j = 0; j < count; j += JOIN * turns) {
                v2f st[JOIN], y[JOIN][2];
                // all on their way at once
#pragma unroll
                for (int e = 0; e < JOIN; e++) {
                    st[e] = v2f{-INFINITY, -1.f};
                    y[e][0] = y[e][1] = v2f{0.f, 0.f};
                    const int at = j + e * turns + turn;
                    if (in && at < count) {
                        const float *p = mine + (size_t)(2 * at + (at == 0)) * slot_size;
                        st[e] = slot_get(p);
                        y[e][0] = slot_get(p + 2 + ch);
                        y[e][1] = slot_get(p + 4 + ch);
                    }
                }
                float to = top;
#pragma unroll
                for (int e = 0; e < JOIN; e++) to = fmaxf(to, st[e][0]);
                const float base = to == -INFINITY ? 0.f : to, old = __builtin_amdgcn_exp2f(top - base);
                sum = sum < 0.f ? sum : sum * old;
                v *= old;
                top = to;
#pragma unroll
                for (int e = 0; e < JOIN; e++) {
                    if (j + e * turns >= count) break;
                    const float f = __builtin_amdgcn_exp2f(st[e][0] - base);
                    if (!(st[e][1] < 0.f)) sum = (sum < 0.f ? 0.f : sum) + st[e][1] * f;
                    v += v4f{y[e][0][0], y[e][0][1], y[e][1][0], y[e][1][1]} * f;
                }
            }
            if (turns > 1) {                // (one round then)
                float *p = lds.o + 8 * tid;
                p[0] = top; p[1] = sum;
                *reinterpret_cast<v4f *>(p + 4) = v;
                __syncthreads();
            }
            if (turn > 0 || !in) continue;
            for (int t = 1; t < turns; t++) {
                const float *p = lds.o + 8 * (tid + t * quads);
                const float to = fmaxf(top, p[0]), base = to == -INFINITY ? 0.f : to;
                const float f0 = __builtin_amdgcn_exp2f(top - base), f1 = __builtin_amdgcn_exp2f(p[0] - base);
                if (!(p[1] < 0.f)) sum = (sum < 0.f ? 0.f : sum * f0) + p[1] * f1;
                else if (!(sum < 0.f)) sum *= f0;
                v = v * f0 + *reinterpret_cast<const v4f *>(p + 4) * f1;
                top = to;
            }
            if (sum < 0.f) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) store_one(op + (size_t)(4 * quad + e) * a.S, v[e] / sum);
            if (lse && ch == 0) lse[out_of(u.col, head0 + h, 1)] = (top + __builtin_amdgcn_logf(sum)) * LN2;
        }
        __syncthreads();
    }
}

// Counts of workgroups that have left a slot; every launch leaves zeros.  (Launches follow one another on the library's stream.)
__device__ unsigned g_arrived[MAX_GROUPS];

template <typename T>
int attn_paged(const char *who, const mi355_kv_cache *c, T *o, float *lse, const T *q, const int32_t *seq, const int32_t *pos, int heads, int S,
               int batch, float scale) {
    if (!kv_cache_ok(who, c)) return -1;
    if (!o || !q || !pos) return mi355_fail("%s: NULL pointer", who);
    if (heads == 0) return mi355_fail("%s: no heads", who);
    if (!kv_columns_ok(who, c, heads, S, batch, seq)) return -1;
    if (!(scale > 0.f) || !isfinite(scale * LOG2E)) return mi355_fail("%s: scale must be positive, and finite times log2(e)", who);
    const size_t units = (size_t)S * batch * heads;
    if (units > 0xffffff) return mi355_fail("%s: %zu heads of columns (at most 2^24 - 1)", who, units);
    // tiles are counted in 32 bits: columns that could have more go in several launches
    const int group = heads / c->kv_heads, parts = (int)ceil_div(group, HEADS), cols = S * batch;
    const size_t column = (ceil_div((size_t)c->max_pages * c->page, Tile<T, 1>::POSITIONS) + BEGIN) * c->kv_heads;
    constexpr size_t COUNT = 0x7fffff00;
    if (column > COUNT)
        return mi355_fail("%s: max_pages * page * kv_heads = %.0f is more tiles than 2^31 - 256", who, (double)c->max_pages * c->page * c->kv_heads);
    if (!mi355_ready(who)) return -1;
    static unsigned *arrived = nullptr;
    if (!arrived) HIP_OK(hipGetSymbolAddress((void **)&arrived, HIP_SYMBOL(g_arrived)));
    const int heads_of = (int)ceil_div(group, parts);
    const bool lengthy = sqrt((double)c->max_pages * c->page / Tile<T, 1>::POSITIONS * heads_of) * PIECE > grain(heads_of);
    const size_t at_once = COUNT / column, most = 2 * g_ctx.num_cu < MAX_GROUPS ? 2 * g_ctx.num_cu : MAX_GROUPS;
    auto go = [&](auto blocks) {
        constexpr int HDB = decltype(blocks)::value;
        float *slots = (float *)mi355_ws(most * 2 * HEADS * (HDB * 32 + 2) * sizeof(float));
        if (!slots) return -1;
        for (size_t c0 = 0; c0 < (size_t)cols; c0 += at_once)
            for (int p0 = 0; p0 < parts; p0 += most / 8) {
                const size_t n = cols - c0 < at_once ? cols - c0 : at_once, useful = ceil_div(n * column, GRAIN);
                const int now = parts - p0 < (int)most / 8 ? parts - p0 : (int)most / 8;
                // workgroups of a part: of several, a multiple of 8
                const size_t room = now == 1 ? most : most / (8 * now) * 8;
                const size_t each = useful < room ? (now == 1 ? useful : ceil_div(useful, 8) * 8) : room;
                const PagedArgs a = {*c, seq, pos, heads, S, (int)c0, (int)n, group, c->max_pages * c->page, p0, now, lengthy ? g_ctx.num_cu : 0,
                                     scale * LOG2E, slots, arrived};
                attn_paged_kernel<T, HDB><<<(unsigned)(each * now), 256, 0, g_ctx.stream>>>(o, lse, q, a);
                LAUNCH_OK(who);
            }
        return 0;
    };
    if (c->hd <= 32) return go(std::integral_constant<int, 1>());
    if (c->hd <= 64) return go(std::integral_constant<int, 2>());
    if (c->hd <= 96) return go(std::integral_constant<int, 3>());
    return go(std::integral_constant<int, 4>());
}

}  // namespace

MI355_API int mi355_attn_paged_dev(const mi355_kv_cache *cache, float *o, float *lse, const float *q, const int32_t *seq, const int32_t *pos, int heads,
                                   int S, int batch, float scale) {
    return attn_paged<float>("attn_paged", cache, o, lse, q, seq, pos, heads, S, batch, scale);
}
MI355_API int mi355_attn_paged_bf16_dev(const mi355_kv_cache *cache, uint16_t *o, float *lse, const uint16_t *q, const int32_t *seq, const int32_t *pos,
                                        int heads, int S, int batch, float scale) {
    return attn_paged<bf16_t>("attn_paged_bf16", cache, o, lse, q, seq, pos, heads, S, batch, scale);
}
