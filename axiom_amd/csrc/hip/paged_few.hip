// Attention over a paged cache for few rows: tokens of sequences that are being written.
//
// Bound by how fast the cache comes in, and for 4 bits by vector instructions.  16 rows (the new tokens of all query heads that share keys, token by token) meet one head of keys, whose 32-key tiles are
// shared out twice: over workgroups, `splits` ranges, and over the eight waves of each (four, where there are at most four tiles), in turn.  A lane loads a quarter of two keys' rows and of the same values' rows, straight
// from their pages, with the next tile's under way meanwhile and the entries of the table for the one after that, which are checked only when they are used:
//   S^T tiles  A = keys from registers (their numbers are f16 exactly, one term; the columns of a lane are neighbours, and the queries' columns lie likewise), B = the queries' two terms
//   softmax    online, in log2 units, as in attn_fwd.hip; a lane owns query (l & 15) and keys 16 t + 4 (l >> 4) + 0..3
//   O^T tiles  A = V^T by transposing reads of an LDS block of the wave's own, B = the probabilities where the score tiles left them, two terms
// so a product of the fp32 ones is two of f16 terms.  Waves meet in LDS, ranges in memory, where the last workgroup to arrive adds them in order: one launch, the same bits whoever is last.
//
// One token over 500 int8 keys, 16 heads, 4 of keys, of 64: 7.8 us (9.2 with four waves and ranges); of 32 sequences over up to 4096, 32 heads, 8 of keys, of 128 49 us, 4.3 TB/s of cache (53 with four waves); equal ones of 8192 5.4
// TB/s; two tokens of 8 over up to 32768 of 4 bits, 64 heads, 8 of keys 62 us.  Entries checked where they are read, which waits for all that is under way: 73 instead of 53, and 87 instead of 63.
#include <algorithm>

#include "attn_launch.h"
#include "attn_tiles.h"
#include "paged.h"

namespace {
using namespace axhip;

constexpr int SPLITS_MOST = PAGED_SPLITS, ROWS = 16;

template <int DK, int WAVES>
struct FewGeom {
    using B = Block<DK, 32>;
    static constexpr int PIECES = DK / 16;                       // a lane's output in pieces of four
    static constexpr int FACTORS_AT = B::PLANE, BLOCK = FACTORS_AT + 256;
    static constexpr int JOIN_AT = 0, ML_AT = WAVES * PIECES * 1024;   // of the waves: pieces [64] v4f, then maxima and sums [2][16]
    static constexpr int BLOCKS = WAVES * BLOCK, JOINED = ML_AT + WAVES * 128, RANGES = SPLITS_MOST * ROWS * 8;
    static constexpr int MOST = BLOCKS > JOINED ? BLOCKS : JOINED, FLAGS_AT = MOST > RANGES ? MOST : RANGES;   // a word a wave: the rows whose sums are not finite; then who is last
    static constexpr int SMEM = FLAGS_AT + 4 * WAVES + 16;
    static_assert(BLOCK % 256 == 0 && SMEM <= 80 * 1024, "LDS");
    static constexpr int PART = PIECES * 256 + 2 * ROWS;         // floats that a range leaves in memory
};

// A lane's quarter of a row as words, in the widest loads that its place allows
template <int WORDS>
struct Quarter {
    static constexpr int WIDE = WORDS % 4 == 0 ? 4 : WORDS % 2 == 0 ? 2 : 1;
    unsigned w[WORDS];
    template <bool PAD>
    __device__ __forceinline__ void load(const unsigned char *quarter, int part, int row_bytes) {
#pragma unroll
        for (int i = 0; i < WORDS; i += WIDE) {
            typedef unsigned wide __attribute__((ext_vector_type(WIDE)));
            const int at = 4 * (part * WORDS + i);
            if (PAD && at >= row_bytes) {
#pragma unroll
                for (int e = 0; e < WIDE; e++) w[i + e] = 0;
            } else if constexpr (WIDE == 1) {
                w[i] = *reinterpret_cast<const unsigned *>(quarter + 4 * i);
            } else {
                const wide v = *reinterpret_cast<const wide *>(quarter + 4 * i);
#pragma unroll
                for (int e = 0; e < WIDE; e++) w[i + e] = v[e];
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = 0;
    }
};

// Columns 8 s .. 8 s + 7 of a lane's quarter as f16
template <int DK, int TYPE, int WORDS>
__device__ __forceinline__ v4i eight_halves(const Quarter<WORDS> &x, int s, int part, unsigned scales, int top) {
    if constexpr (TYPE == AXHIP_KV_F16) return v4i{(int)x.w[4 * s], (int)x.w[4 * s + 1], (int)x.w[4 * s + 2], (int)x.w[4 * s + 3]};
    if constexpr (TYPE == AXHIP_KV_I8) {
        v4i h;
        int a, b;
        kv_bytes(x.w[2 * s], a, b);
        h[0] = a;
        h[1] = b;
        kv_bytes(x.w[2 * s + 1], a, b);
        h[2] = a;
        h[3] = b;
        return h;
    }
    if constexpr (TYPE == AXHIP_KV_MX4) return kv_nibbles(x.w[s], mx4_up(scales, top, (part * (DK / 4) + 8 * s) / 32));
}

template <int DK, int TYPE, bool PAD, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) k_paged_few(PagedArgs a, PagedFewGrid grid) {
    using G = FewGeom<DK, WAVES>;
    using B = typename G::B;
    using T = KvType<TYPE>;
    constexpr int KS = DK / 32, PIECES = G::PIECES, MINE = (PIECES + WAVES - 1) / WAVES, WORDS = DK * T::BITS / 128;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const KvPages &kv = a.pages;
    const AttnArgs &at = a.attn;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 15, part = lane >> 4;
    // Ranges of one set of rows follow each other, so that they go to different XCDs; the sequences' second sets of rows, which few may have, come behind all first ones, so that those do.
    const unsigned local = blockIdx.x / (unsigned)grid.splits, split = blockIdx.x - local * (unsigned)grid.splits, each = (unsigned)grid.here * (unsigned)kv.heads, of_b = local % each;
    const int rt = (int)(local / each), b = grid.first + (int)(of_b / (unsigned)kv.heads), hk = (int)(of_b % (unsigned)kv.heads);
    const int64_t unit = (int64_t)grid.first * kv.heads * grid.row_tiles + local;
    const KvSeq seq = kv_seq(kv, b);
    const int64_t rows = (int64_t)at.G * seq.n;
    if ((int64_t)rt * ROWS >= rows || rows > grid.most) return;
    const int r = rt * ROWS + frow;
    const bool valid = r < rows;
    const int i = (int)((valid ? r : (int)rows - 1) / at.G), head = hk * at.G + (valid ? r : (int)rows - 1) - i * at.G;
    PagedRow row = paged_row(a, seq, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0;
    // what the rows see together: they go up with their positions
    const PagedRow low = paged_row(a, seq, rt * ROWS / at.G), high = paged_row(a, seq, (int)(min((int64_t)rt * ROWS + ROWS, rows) - 1) / at.G);
    const PagedTiles tiles = paged_tiles_of(a, low.begin, high.end, 5);
    const int t_begin = (int)((unsigned)tiles.all * split / (unsigned)grid.splits), t_end = (int)((unsigned)tiles.all * (split + 1) / (unsigned)grid.splits);
    const float slope2 = at.slopes ? at.slopes[head] * at.bias2 : 0.0f;

    unsigned char *const mine = lds + wave * G::BLOCK;
    float *const factors = reinterpret_cast<float *>(mine + G::FACTORS_AT);
    const unsigned base = lds_address(mine);

    // keys frow and 16 + frow of a tile, and the entries of the table for those of the next
    Quarter<WORDS> kq[2], vq[2];
    unsigned ks[2], vs[2];
    int entry[2];
    bool here[2];
    const int32_t *const entries = kv.table + (int64_t)b * kv.table_ld;
    // where this lane's quarter of row zero of a page zero is, and the scale of that row
    const unsigned char *const k0 = kv.k + kv_row_at(kv, 0, hk, 0) + part * WORDS * 4;
    const unsigned char *const s0 = kv.k_scale + kv_scale_at(kv, 0, hk, 0);
    const int64_t to_v = kv.v - kv.k, to_v_scale = kv.v_scale - kv.k_scale;
    auto pos_of = [&](int n, int t) { return tiles.tile(n) * 32 + 16 * t + frow; };
    auto look = [&](int n) {
#pragma unroll
        for (int t = 0; t < 2; t++) entry[t] = entries[(unsigned)min(pos_of(n, t), high.end - 1) >> kv.shift];
    };
    auto fetch = [&](int n) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int pos = pos_of(n, t);
            here[t] = pos < high.end && kv_is_page(kv, entry[t]);
            ks[t] = vs[t] = 0;
            if (here[t]) {
                const unsigned in_page = (unsigned)pos & ((1u << kv.shift) - 1);
                const unsigned char *const row = k0 + ((uint64_t)(unsigned)entry[t] * kv.page_bytes + __umul24(in_page, (unsigned)kv.row_bytes));
                const unsigned char *const scale = s0 + ((uint64_t)(unsigned)entry[t] * kv.page_scales + 4 * in_page);
                ks[t] = *reinterpret_cast<const unsigned *>(scale);
                vs[t] = *reinterpret_cast<const unsigned *>(scale + to_v_scale);
                kq[t].template load<PAD>(row, part, kv.row_bytes);
                vq[t].template load<PAD>(row + to_v, part, kv.row_bytes);
            }
        }
    };
    // (where there is no page the numbers of an earlier tile stay, which are finite, under a factor of zero)
#pragma unroll
    for (int t = 0; t < 2; t++) {
        kq[t].clear();
        vq[t].clear();
    }
    int n = t_begin + wave;
    if (n < t_end) {
        look(n);
        fetch(n);
        if (n + WAVES < t_end) look(n + WAVES);
    }
    v4i qf[KS][2];                                   // step s: columns part * DK / 4 + 8 s .. + 7 of this lane's query
    float q_down;
    {
        const float *q = at.Q + ((int64_t)seq.first + i) * at.ldq + (int64_t)head * kv.dk + part * (DK / 4);
        float x[KS][8];
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                v4f v = {0.f, 0.f, 0.f, 0.f};
                if (live && (!PAD || part * (DK / 4) + 8 * s + 4 * h < kv.dk)) v = *reinterpret_cast<const v4f *>(q + 8 * s + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; e++) x[s][4 * h + e] = v[e] * at.q_up;
            }
        q_down = cut_row(x, most_of_parts(most_of(x)), qf);
    }
    v4f acc[PIECES];
#pragma unroll
    for (int d = 0; d < PIECES; d++) acc[d] = v4f{0.f, 0.f, 0.f, 0.f};
    float ref = ATTN_LOWEST, l_run = 0.0f;           // acc is 2^VALUE_BIAS times the sum
    const float one = hidden_one();
    const bool plain = at.cap == 0.0f && !at.slopes;
    const float down = plain ? q_down : 1.0f;        // what is left to the score in the exponential's multiply-add
    const unsigned column_at = B::column_place16(lane) + base;

    for (; n < t_end; n += WAVES) {
        const int kt0 = tiles.tile(n) * 32;
        order_in_wave();                             // the last tile has been read
        int top_k[2], top_v[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            top_k[t] = TYPE == AXHIP_KV_MX4 ? mx4_top(ks[t]) : 0;
            top_v[t] = TYPE == AXHIP_KV_MX4 ? mx4_top(vs[t]) : 0;
            if (part == 0) {
                factors[16 * t + frow] = kv_factor<TYPE>(ks[t]);
                factors[32 + 16 * t + frow] = kv_factor<TYPE>(vs[t]) * T::VALUE_UP * VALUES_DOWN;
            }
        }
        const uint64_t gone0 = __builtin_amdgcn_ballot_w64(!here[0]), gone1 = __builtin_amdgcn_ballot_w64(!here[1]);
        const unsigned gone = ((unsigned)gone0 & 0xffffu) | (unsigned)gone1 << 16;
        v4f s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const v8h f = __builtin_bit_cast(v8h, (eight_halves<DK, TYPE, WORDS>(kq[t], k, part, ks[t], top_k[t])));
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, __builtin_bit_cast(v8h, qf[k][1]), s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, __builtin_bit_cast(v8h, qf[k][0]), s[t], 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < KS; k++)
                write_chunk(base + B::at(16 * t + frow, part * KS + k), eight_halves<DK, TYPE, WORDS>(vq[t], k, part, vs[t], top_v[t]));
        }
        order_in_wave();
        if (n + WAVES < t_end) {
            fetch(n + WAVES);
            if (n + 2 * WAVES < t_end) look(n + 2 * WAVES);
        }
        v4f vf[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const v4f kf = *reinterpret_cast<const v4f *>(factors + 16 * t + 4 * part);
            vf[t] = *reinterpret_cast<const v4f *>(factors + 32 + 16 * t + 4 * part);
            s[t] *= kf;
            if (!plain) s[t] *= q_down;
        }
        if (__builtin_expect(at.cap > 0.0f, 0)) {
            float big = 0.0f;
#pragma unroll
            for (int v = 0; v < 8; v++) big = fmaxf(big, __builtin_fabsf(s[v >> 2][v & 3]));
            if (__builtin_amdgcn_ballot_w64(!(big < at.cap_near)))
#pragma unroll
                for (int v = 0; v < 8; v++) s[v >> 2][v & 3] = capped(at, s[v >> 2][v & 3]).score;
            else
#pragma unroll
                for (int v = 0; v < 8; v++) s[v >> 2][v & 3] = capped_near(at, s[v >> 2][v & 3]).score;
        }
        if (__builtin_expect(at.slopes != nullptr, 0)) {
            const float from = (float)(row.p - kt0 - 4 * part);
#pragma unroll
            for (int v = 0; v < 8; v++) s[v >> 2][v & 3] = __builtin_fmaf(-slope2, from - (float)(16 * (v >> 2) + (v & 3)), s[v >> 2][v & 3]);
        }
        // (all rows see a tile before the first one's end and, where it is none of the first tokens only, behind the last one's beginning; rows that see nothing are not written)
        const bool partly = gone != 0 || kt0 + 32 > low.end || (kt0 < high.begin && kt0 + 32 > a.sinks);
        if (__builtin_expect(partly, 0)) {
            const int end = row.end - kt0 - 4 * part, begin = row.begin - kt0 - 4 * part, first = a.sinks - kt0 - 4 * part;
            const unsigned none = gone >> (4 * part);
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const int j = 16 * (v >> 2) + (v & 3);
                if (j >= end || (j < begin && j >= first) || ((none >> j) & 1)) s[v >> 2][v & 3] = -INFINITY;
            }
        }
        float x[8], most, l_blk;
        auto weigh = [&]() {
            most = l_blk = 0.0f;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v >> 2][v & 3], down, -ref));
                l_blk += p;
                x[v] = p * vf[v >> 2][v & 3];
                most = fmaxf(most, x[v]);
            }
        };
        weigh();
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > ROOM) != 0, 0)) {          // (always for the first finite scores)
            most = most_of_parts(most);
            float top = -INFINITY;
#pragma unroll
            for (int v = 0; v < 8; v++) top = fmaxf(top, __builtin_fmaf(s[v >> 2][v & 3], down, __builtin_amdgcn_logf(vf[v >> 2][v & 3])));
            top = most_of_parts(top) - (float)LARGEST;
            const float next = most > ROOM ? fmaxf(ref, top) : ref, alpha = __builtin_amdgcn_exp2f(ref - next);
            l_run = scaled(l_run, ref - next);
            ref = next;
#pragma unroll
            for (int d = 0; d < PIECES; d++) acc[d] *= alpha;
            weigh();
        }
        l_run += l_blk;
        v4i pf[2];
        cut_scaled(x, one, pf);
        // (columns are read two pieces ahead)
        v4i f[3];
        f[0] = B::columns16(column_at, 0, 0);
        if (PIECES > 1) f[1] = B::columns16(column_at, 1, 0);
        __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
        for (int d = 0; d < PIECES; d++) {
            if (d + 2 < PIECES) f[(d + 2) % 3] = B::columns16(column_at, d + 2, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, f[d % 3]), __builtin_bit_cast(v8h, pf[1]), acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, f[d % 3]), __builtin_bit_cast(v8h, pf[0]), acc[d], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0x6);
        }
    }

    // ---- the waves' parts together ----
    __syncthreads();                                 // the blocks have been read
    v4f *const parts = reinterpret_cast<v4f *>(lds + G::JOIN_AT);
    float *const ml = reinterpret_cast<float *>(lds + G::ML_AT);
    const float l_wave = over_parts(l_run, [](float x, float y) { return x + y; });
#pragma unroll
    for (int d = 0; d < PIECES; d++) parts[(wave * PIECES + d) * 64 + lane] = acc[d] * two_to(-T::VALUE_BIAS);
    if (part == 0) {
        ml[wave * 32 + frow] = ref;
        ml[wave * 32 + ROWS + frow] = l_wave;
    }
    __syncthreads();
    float m_all = ATTN_LOWEST, l_all = 0.0f, weight[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; w++) m_all = fmaxf(m_all, ml[w * 32 + frow]);
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        weight[w] = __builtin_amdgcn_exp2f(ml[w * 32 + frow] - m_all);
        l_all += scaled(ml[w * 32 + ROWS + frow], ml[w * 32 + frow] - m_all);
    }
    v4f out[MINE];                                   // this wave's pieces: wave, wave + 4
#pragma unroll
    for (int d = 0; d < MINE; d++) {
        out[d] = v4f{0.f, 0.f, 0.f, 0.f};
        if (wave + WAVES * d < PIECES)
#pragma unroll
            for (int w = 0; w < WAVES; w++) out[d] += parts[(w * PIECES + wave + WAVES * d) * 64 + lane] * weight[w];
    }
    int *const flags = reinterpret_cast<int *>(lds + G::FLAGS_AT);
    if (grid.splits > 1) {
        // The ranges meet in memory, as those of attn_few.hip do: device-scope accesses throughout; the wait completes a thread's stores before the barrier, the barrier orders
        // them before thread 0's increment.
        typedef float v2f __attribute__((ext_vector_type(2)));
        float *to_memory = grid.parts + (unit * grid.splits + split) * G::PART;
#pragma unroll
        for (int d = 0; d < MINE; d++) {
            if (wave + WAVES * d >= PIECES) break;
            int64_t *to = reinterpret_cast<int64_t *>(to_memory + ((wave + WAVES * d) * 64 + lane) * 4);
            __hip_atomic_store(to, __builtin_bit_cast(int64_t, v2f{out[d][0], out[d][1]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(to + 1, __builtin_bit_cast(int64_t, v2f{out[d][2], out[d][3]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (wave == 0 && part == 0)
            __hip_atomic_store(reinterpret_cast<int64_t *>(to_memory + PIECES * 256 + 2 * frow), __builtin_bit_cast(int64_t, v2f{m_all, l_all}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0) flags[WAVES] = __hip_atomic_fetch_add(grid.arrivals + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == grid.splits - 1;
        __syncthreads();
        if (!flags[WAVES]) return;
        const float *theirs = grid.parts + unit * grid.splits * G::PART;
        auto read = [&](int64_t from) {
            return __builtin_bit_cast(v2f, __hip_atomic_load(reinterpret_cast<const int64_t *>(theirs + from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        // Every read is a trip to memory, so they go out together: maxima and sums by groups of 16 lanes, and AHEAD ranges' outputs at a time.
        constexpr int AHEAD = 8, GROUPS = 4 * WAVES, EACH = SPLITS_MOST / GROUPS;
        v2f *const both = reinterpret_cast<v2f *>(lds + G::JOIN_AT) + frow;
        v2f here[EACH];
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const int from = (int)(threadIdx.x >> 4) + GROUPS * k;
            if (from < grid.splits) here[k] = read((int64_t)from * G::PART + PIECES * 256 + 2 * frow);
        }
        v4f x[AHEAD][MINE];
        auto outputs = [&](int s0) {
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (s0 + k >= grid.splits) break;
#pragma unroll
                for (int d = 0; d < MINE; d++) {
                    if (wave + WAVES * d >= PIECES) break;
                    const int64_t from = (int64_t)(s0 + k) * G::PART + ((wave + WAVES * d) * 64 + lane) * 4;
                    const v2f p = read(from), q = read(from + 2);
                    x[k][d] = v4f{p[0], p[1], q[0], q[1]};
                }
            }
        };
        outputs(0);
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const int from = (int)(threadIdx.x >> 4) + GROUPS * k;
            if (from < grid.splits) both[ROWS * from] = here[k];
        }
        __syncthreads();
        m_all = ATTN_LOWEST;
        for (int from = 0; from < grid.splits; from++) m_all = fmaxf(m_all, both[ROWS * from][0]);
        l_all = 0.0f;
#pragma unroll
        for (int d = 0; d < MINE; d++) out[d] = v4f{0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < grid.splits; s0 += AHEAD) {
            if (s0 > 0) outputs(s0);
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (s0 + k >= grid.splits) break;
                const v2f ml_here = both[ROWS * (s0 + k)];
                const float w = __builtin_amdgcn_exp2f(ml_here[0] - m_all);
                l_all += scaled(ml_here[1], ml_here[0] - m_all);
#pragma unroll
                for (int d = 0; d < MINE; d++)
                    if (wave + WAVES * d < PIECES) out[d] += x[k][d] * w;
            }
        }
        if (threadIdx.x == 0) __hip_atomic_store(grid.arrivals + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);       // ready for the next launch
    }

    // ---- normalise and write ----
    float seen = l_all * 0.0f;
#pragma unroll
    for (int d = 0; d < MINE; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(out[d][e], 0.0f, seen);
    const uint64_t unfit = __builtin_amdgcn_ballot_w64(live && (!(seen == 0.0f) || l_all == 0.0f));
    if (lane == 0) flags[wave] = (int)((unsigned)(unfit | unfit >> 16 | unfit >> 32 | unfit >> 48) & 0xffffu);
    __syncthreads();
    unsigned again = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) again |= (unsigned)flags[w];
    again = __builtin_amdgcn_readfirstlane(again);
    if (valid && !((again >> frow) & 1)) {
        const float inv = 1.0f / l_all;
        const int64_t to = (int64_t)seq.first + i;
        float *o = at.O + to * at.ldo + (int64_t)head * kv.dk;
#pragma unroll
        for (int d = 0; d < MINE; d++) {
            const int piece = wave + WAVES * d, col = 16 * piece + 4 * part;
            if (piece < PIECES && (!PAD || col < kv.dk)) *reinterpret_cast<v4f *>(o + col) = live ? out[d] * inv : v4f{0.f, 0.f, 0.f, 0.f};
        }
        if (at.L && wave == 0 && part == 0) at.L[to * at.H + head] = live ? (m_all + __builtin_amdgcn_logf(l_all)) * LN2 : -INFINITY;
    }
    int nth = 0;
    for (unsigned rest = again; rest; rest &= rest - 1, nth++) {
        const int n = __builtin_ctz(rest);
        if (nth % WAVES == wave) paged_again<TYPE>(a, b, seq, __builtin_amdgcn_readlane(head, n), __builtin_amdgcn_readlane(i, n), lane);
    }
}

template <int DK, int TYPE, bool PAD, int WAVES>
int launch_few(const PagedArgs &a, PagedFewGrid grid) {
    using G = FewGeom<DK, WAVES>;
    static bool attr_set = false;
    if (!attr_set) {
        AXHIP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(k_paged_few<DK, TYPE, PAD, WAVES>), hipFuncAttributeMaxDynamicSharedMemorySize, G::SMEM), "hipFuncSetAttribute");
        attr_set = true;
    }
    const int64_t of_b = (int64_t)a.pages.heads * grid.row_tiles, units = a.pages.B * of_b;
    if (grid.splits > 1) {
        grid.parts = static_cast<float *>(workspace((size_t)units * grid.splits * G::PART * sizeof(float)));
        grid.arrivals = strip_counters((size_t)units);
        if (!grid.parts || !grid.arrivals) return AXHIP_ERR_ALLOC;
    }
    note_kernel(grid.splits > 1 ? "paged_few_ranges" : "paged_few");
    const int64_t at_once = std::max<int64_t>(1, GRID_MOST / (of_b * grid.splits));      // sequences a launch; (one has at most 2^22 units, of 2^20 heads with 64 rows, and ranges only where there are few)
    for (grid.first = 0; grid.first < a.pages.B; grid.first += (int)at_once) {
        const int64_t left = a.pages.B - grid.first, here = left < at_once ? left : at_once;
        grid.here = (int)here;
        hipLaunchKernelGGL((k_paged_few<DK, TYPE, PAD, WAVES>), dim3((unsigned)(here * of_b * grid.splits)), dim3(64 * WAVES), G::SMEM, kStream, a, grid);
        if (int rc = check_launch("attn_paged")) return rc;
    }
    return AXHIP_OK;
}

template <int DK, int TYPE, int WAVES>
int launch_few(const PagedArgs &a, const PagedFewGrid &grid) {
    return a.pages.dk < DK ? launch_few<DK, TYPE, true, WAVES>(a, grid) : launch_few<DK, TYPE, false, WAVES>(a, grid);
}
template <int DK, int WAVES>
int launch_few(const PagedArgs &a, int type, const PagedFewGrid &grid) {
    return type == AXHIP_KV_F16 ? launch_few<DK, AXHIP_KV_F16, WAVES>(a, grid) : type == AXHIP_KV_I8 ? launch_few<DK, AXHIP_KV_I8, WAVES>(a, grid) : launch_few<DK, AXHIP_KV_MX4, WAVES>(a, grid);
}

}  // namespace

namespace axhip {

int64_t paged_few_splits(int64_t units, int64_t tiles) { return best_splits(units, (tiles + 7) / 8, (tiles + 15) / 16, 2, 1); }

int paged_few(const PagedArgs &a, int type, int rows_most) {
    PagedFewGrid grid = {};
    grid.most = rows_most;
    const int64_t rows = (int64_t)a.attn.G * a.pages.Sq, most = rows < rows_most ? rows : rows_most, tiles = paged_steps_most(a, 5, ROWS);
    grid.row_tiles = (int)((most + ROWS - 1) / ROWS);
    // In how many ranges goes by the sets of rows that there are; where only some of the sequences are this form's, most of those have a single new token.  Where a sequence may have all rows of the
    // call, they are taken to be one token each and the others in full sets: eight single tokens over 4096 int8 keys, 64 heads, 8 of keys, of 128, with Sq = 8 or more 21 us as with Sq = 1, and 38 by the most
    // that each may have.  (Not so for counts between: workgroups that find nothing delay others, and ranges make more of those.  16 tokens of one of 16 sequences and one of each other, 4 bits: 25 instead of 19.)
    const int64_t B = a.pages.B, T = a.pages.T, of_token = (a.attn.G + ROWS - 1) / ROWS, some = std::min(B, T);
    int64_t sets = B * (rows <= rows_most ? grid.row_tiles : of_token);
    if (a.pages.first && rows <= rows_most && T == a.pages.Sq)
        sets = std::min(sets, std::max(some * of_token + (a.attn.G * (T - some) + ROWS - 1) / ROWS, sets / 4));      // (a quarter at least: of what finds nothing, and what it could leave, there is no more than four times)
    grid.splits = (int)paged_few_splits(a.pages.heads * sets, tiles);
    const int waves = tiles > 4 ? 8 : 4;
    auto run = [&](auto width) {
        constexpr int DK = decltype(width)::value;
        return waves == 8 ? launch_few<DK, 8>(a, type, grid) : launch_few<DK, 4>(a, type, grid);
    };
    if (a.pages.dk <= 32) return run(std::integral_constant<int, 32>());
    if (a.pages.dk <= 64) return run(std::integral_constant<int, 64>());
    if (a.pages.dk <= 96) return run(std::integral_constant<int, 96>());
    return run(std::integral_constant<int, 128>());
}

}  // namespace axhip
