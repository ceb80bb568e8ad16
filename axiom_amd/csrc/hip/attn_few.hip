// Attention forward under score rules for few rows: tokens over a cache, short prompts.
//
// Bound by how fast K and V come in.  32 rows (the new tokens of all query heads that share keys, one head after the other) meet one head of keys, and the keys are
// shared out twice: over workgroups, `splits` ranges of a sequence's 32-key tiles, and over the four waves of each, which take its tiles in turn.  A wave brings its own
// tile, whole rows of K and V by 16-byte loads with the next tile in registers meanwhile, cuts it into an LDS block of its own (no barrier until the end) and goes through it as
// the tile kernel does (attn_fwd.hip).  Maxima, sums and outputs of the waves meet in LDS, those of the ranges in memory, where the last workgroup of the rows to arrive adds
// them, in order: one launch, and the same bits whoever is last.
//
// A token of each of 32 sequences over 2048 to 4096 keys, 32 heads, 8 of keys, of 128 takes 169 us, 4.8 TB/s of cache; the matrix core is busy a tenth of the cycles, vector instructions two fifths.
// One token over 500 keys, 16 heads, 4 of keys, of 64: 10.2 us, latency of lengths, keys and the join (15.3 in one range).
#include "attn_launch.h"
#include "attn_tiles.h"

namespace {
using namespace axhip;

constexpr int WAVES = 4, SPLITS_MOST = 64;

template <int DK>
struct FewGeom {
    using B = Block<DK, 32>;
    static constexpr int DT = DK / 32, PIECES = 4 * DT;          // a lane's output in pieces of four
    static constexpr int FACTORS_AT = 2 * B::BYTES, DOCS_AT = FACTORS_AT + 256, BLOCK = DOCS_AT + 256;
    static constexpr int JOIN_AT = 0, ML_AT = WAVES * PIECES * 1024;   // of the waves: pieces [64] v4f, then maxima and sums [2][32]
    static constexpr int BLOCKS = WAVES * BLOCK, JOINED = ML_AT + WAVES * 256;
    static constexpr int FLAGS_AT = BLOCKS > JOINED ? BLOCKS : JOINED;   // a word a wave: the rows whose sums are not finite; then who is last
    static constexpr int SMEM = FLAGS_AT + 4 * WAVES + 16;
    static_assert(BLOCK % 256 == 0 && SMEM <= 160 * 1024, "LDS");
    static constexpr int PART = PIECES * 64 * 4 + 64;            // floats that a range leaves in memory
};

template <int DK, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, (DK <= 64 ? 2 : 1)) k_attn_few(AttnArgs a, FewGrid grid) {
    using G = FewGeom<DK>;
    using B = typename G::B;
    constexpr int KS = DK / 16, DT = DK / 32, PIECES = G::PIECES;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;
    // ranges of one set of rows follow each other, so that they go to different XCDs
    const int64_t unit = blockIdx.x / grid.splits;
    const int split = (int)(blockIdx.x - unit * grid.splits);
    const int64_t bh = unit / grid.row_tiles;
    const int rt = (int)(unit - bh * grid.row_tiles), b = (int)(bh / a.Hkv), hk = (int)(bh - (int64_t)b * a.Hkv), h0 = hk * a.G;
    const int rows = a.G * a.Sq, r = rt * 32 + frow;
    const bool valid = r < rows, docs = a.doc_q != nullptr;
    const int over = (valid ? r : rows - 1) / a.Sq, head = h0 + over, i = (valid ? r : rows - 1) - over * a.Sq;
    AttnRow row = attn_row(a, b, head, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0;
    const RowsSeen mine = same_for_wave(rows_seen(row));
    const int last = mine.last, sure = mine.sure, d_low = mine.low, d_high = mine.high;
    const int all = (last + 31) / 32, t_begin = (int)((int64_t)all * split / grid.splits), t_end = (int)((int64_t)all * (split + 1) / grid.splits);

    const float *Kb = a.K + (int64_t)b * a.kv_rows * a.ldk + (int64_t)hk * a.dk, *Vb = a.V + (int64_t)b * a.kv_rows * a.ldv + (int64_t)hk * a.dk;
    unsigned char *const at = lds + wave * G::BLOCK;
    float *const row_factors = reinterpret_cast<float *>(at + G::FACTORS_AT);
    const unsigned base = lds_address(at);
    using S = Stage<DK, 32, 1, PAD>;
    S ks, vs;
    int doc_here = -1;
    auto load = [&](int t) {
        const int64_t k0 = (int64_t)t * 32;
        const int end = last - 1 - (int)k0;          // rows past it are read as it
        const int l = (int)afresh(lane);
        ks.load(Kb + k0 * a.ldk, a.ldk, end, S::place(0, l, a.ldk), l, a.dk);
        vs.load(Vb + k0 * a.ldv, a.ldv, end, S::place(0, l, a.ldv), l, a.dk);
        if (docs) doc_here = frow <= end ? a.doc_k[(int64_t)b * a.Sk + k0 + frow] : -1;
    };
    int t = t_begin + wave;
    if (t < t_end) load(t);
    v4i qf[KS][2];
    float q_down;
    {
        const float *q = a.Q + ((int64_t)b * a.Sq + i) * a.ldq + (int64_t)head * a.dk;
        float x[KS][8];
        load_row<PAD, 2>(x, q, live, fhalf, a.dk);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] *= a.q_up;
        const float most = most_of(x);
        q_down = cut_row(x, fmaxf(most, __shfl_xor(most, 32, 64)), qf);
    }
    v16f acc[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[d][v] = 0.0f;
    float ref = ATTN_LOWEST, l_run = 0.0f;           // as in the tile kernel: acc is 2^BIAS times the sum
    const float one = hidden_one();

    const unsigned row_at = B::row_place(lane) + base, column_at = B::column_place(lane) + base + B::BYTES;
    for (; t < t_end; t += WAVES) {
        const int kt0 = t * 32;
        bool partly = kt0 + 32 > sure, meets = true;
        if (docs) {
            meets = __builtin_amdgcn_ballot_w64(doc_here >= d_low && doc_here <= d_high) != 0;
            partly |= __builtin_amdgcn_ballot_w64(doc_here != d_low) != 0 || d_low != d_high;
        }
        order_in_wave();                             // the last tile has been read
        if (meets) {
            const int l = (int)afresh(lane);
            const typename S::Place place = S::place(0, l, 0);
            ks.put(base, base + G::FACTORS_AT, place, l, 1.0f, a.dk);
            vs.put(base + B::BYTES, base + G::FACTORS_AT + 128, place, l, VALUES_UP, a.dk, VALUES_DOWN);
            if (docs && lane < 32) reinterpret_cast<int *>(at + G::DOCS_AT)[lane] = doc_here;
        }
        order_in_wave();
        if (t + WAVES < t_end) load(t + WAVES);
        if (!meets) continue;
        const unsigned row_place = afresh(row_at), column_place = afresh(column_at);
        v16f s;
#pragma unroll
        for (int v = 0; v < 16; v++) s[v] = 0.0f;
        products<KS>(
            [&](int k, v4i (&f)[2]) {
                f[1] = B::rows(row_place, k, 1);
                f[0] = B::rows(row_place, k, 0);
            },
            [&](int k, const v4i (&f)[2]) { s = mfma_cut(f, qf[k], s); });
        auto factors = [&](int what, int g) { return *reinterpret_cast<const v4f *>(row_factors + what * 32 + 8 * g + 4 * fhalf); };
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const v4f f = factors(0, g);
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * g + e] *= f[e] * q_down;
        }
        if (a.cap > 0.0f) {
            float big = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; v++) big = fmaxf(big, __builtin_fabsf(s[v]));
            if (__builtin_amdgcn_ballot_w64(!(big < a.cap_near)))
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] = capped(a, s[v]).score;
            else
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] = capped_near(a, s[v]).score;
        }
        if (a.slopes) {
            const float from = (float)(row.p - kt0 - 4 * fhalf);
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = __builtin_fmaf(-row.slope2, __builtin_fabsf(from - (float)(8 * (v >> 2) + (v & 3))), s[v]);
        }
        if (partly) {
            const int end = row.end - kt0 - 4 * fhalf;
#pragma unroll
            for (int v = 0; v < 16; v++)
                if (8 * (v >> 2) + (v & 3) >= end) s[v] = -INFINITY;
            if (docs)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const v4i d = *reinterpret_cast<const v4i *>(at + G::DOCS_AT + 4 * (8 * g + 4 * fhalf));
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (d[e] != row.doc) s[4 * g + e] = -INFINITY;
                }
        }
        v16f x;
        float most, l_blk;
        auto weigh = [&]() {
            most = l_blk = 0.0f;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f f = factors(1, g);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int v = 4 * g + e;
                    const float p = __builtin_amdgcn_exp2f(s[v] - ref);
                    l_blk += p;
                    x[v] = p * f[e];
                    most = fmaxf(most, x[v]);
                }
            }
        };
        weigh();
        if (__builtin_amdgcn_ballot_w64(most > ROOM)) {
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f f = factors(1, g);
#pragma unroll
                for (int e = 0; e < 4; e++) top = fmaxf(top, s[4 * g + e] + __builtin_amdgcn_logf(f[e]));
            }
            top = fmaxf(top, __shfl_xor(top, 32, 64)) - (float)LARGEST;
            const float next = most > ROOM ? fmaxf(ref, top) : ref, alpha = __builtin_amdgcn_exp2f(ref - next);
            l_run = scaled(l_run, ref - next);
            ref = next;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[d][v] *= alpha;
            weigh();
        }
        l_run += l_blk;
        v4i pf[2][2];
        cut_scaled(x, 0, one, pf[0]);
        cut_scaled(x, 1, one, pf[1]);
        products<2 * DT>(
            [&](int n, v4i (&f)[2]) {
                f[1] = B::columns(column_place, 16 * (n / DT), n % DT, 1);
                f[0] = B::columns(column_place, 16 * (n / DT), n % DT, 0);
            },
            [&](int n, const v4i (&f)[2]) { acc[n % DT] = mfma_cut(f, pf[n / DT], acc[n % DT]); });
    }

    // ---- the waves' parts together ----
    __syncthreads();                                 // the blocks have been read
    v4f *const part = reinterpret_cast<v4f *>(lds + G::JOIN_AT);
    float *const ml = reinterpret_cast<float *>(lds + G::ML_AT);
    const float l_wave = l_run + __shfl_xor(l_run, 32, 64);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            part[(wave * PIECES + 4 * d + g) * 64 + lane] = v4f{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]} * two_to(-BIAS);
    if (fhalf == 0) {
        ml[wave * 64 + frow] = ref;
        ml[wave * 64 + 32 + frow] = l_wave;
    }
    __syncthreads();
    float m_all = ATTN_LOWEST, l_all = 0.0f, weight[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; w++) m_all = fmaxf(m_all, ml[w * 64 + frow]);
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        weight[w] = __builtin_amdgcn_exp2f(ml[w * 64 + frow] - m_all);
        l_all += scaled(ml[w * 64 + 32 + frow], ml[w * 64 + frow] - m_all);
    }
    v4f out[DT];                                     // this wave's pieces: wave, wave + 4, ...
#pragma unroll
    for (int n = 0; n < DT; n++) {
        out[n] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) out[n] += part[(w * PIECES + wave + 4 * n) * 64 + lane] * weight[w];
    }
    int *const flags = reinterpret_cast<int *>(lds + G::FLAGS_AT);
    if (grid.splits > 1) {
        // The ranges meet in memory: parts, counter and the reads below are device-scope accesses (the workgroups run on XCDs with an L2 each); the wait
        // completes a thread's stores before the barrier, the barrier orders them before thread 0's increment.
        typedef float v2f __attribute__((ext_vector_type(2)));
        float *mine = grid.parts + (unit * grid.splits + split) * G::PART;
#pragma unroll
        for (int n = 0; n < DT; n++) {
            int64_t *to = reinterpret_cast<int64_t *>(mine + ((wave + 4 * n) * 64 + lane) * 4);
            __hip_atomic_store(to, __builtin_bit_cast(int64_t, v2f{out[n][0], out[n][1]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(to + 1, __builtin_bit_cast(int64_t, v2f{out[n][2], out[n][3]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (wave == 0 && fhalf == 0)
            __hip_atomic_store(reinterpret_cast<int64_t *>(mine + PIECES * 256 + 2 * frow), __builtin_bit_cast(int64_t, v2f{m_all, l_all}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (threadIdx.x == 0) flags[WAVES] = __hip_atomic_fetch_add(grid.arrivals + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == grid.splits - 1;
        __syncthreads();
        if (!flags[WAVES]) return;
        const float *theirs = grid.parts + unit * grid.splits * G::PART;
        auto read = [&](int64_t from) {
            return __builtin_bit_cast(v2f, __hip_atomic_load(reinterpret_cast<const int64_t *>(theirs + from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        };
        // Every read is a trip to memory, so they go out together: maxima and sums by eight groups of 32 lanes, then AHEAD ranges' outputs at a time.  (5 tokens of 4 sequences over 9578
        // keys, 2 heads of keys of 32, in 64 ranges: 39 us with four at a time and the maxima one after the other, 23 so.)
        static_assert(SPLITS_MOST == 64 && G::JOINED >= 64 * 256, "LDS for the maxima and sums of all ranges");
        v2f *const both = reinterpret_cast<v2f *>(lds + G::JOIN_AT) + frow;
        v2f here[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int s = (int)(threadIdx.x >> 5) + 8 * k;
            if (s < grid.splits) here[k] = read((int64_t)s * G::PART + PIECES * 256 + 2 * frow);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int s = (int)(threadIdx.x >> 5) + 8 * k;
            if (s < grid.splits) both[32 * s] = here[k];
        }
        __syncthreads();
        m_all = ATTN_LOWEST;
        for (int s = 0; s < grid.splits; s++) m_all = fmaxf(m_all, both[32 * s][0]);
        l_all = 0.0f;
#pragma unroll
        for (int n = 0; n < DT; n++) out[n] = v4f{0.f, 0.f, 0.f, 0.f};
        constexpr int AHEAD = 8;
        for (int s0 = 0; s0 < grid.splits; s0 += AHEAD) {
            v4f x[AHEAD][DT];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (s0 + k >= grid.splits) break;
#pragma unroll
                for (int n = 0; n < DT; n++) {
                    const int64_t from = (int64_t)(s0 + k) * G::PART + ((wave + 4 * n) * 64 + lane) * 4;
                    const v2f p = read(from), q = read(from + 2);
                    x[k][n] = v4f{p[0], p[1], q[0], q[1]};
                }
            }
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (s0 + k >= grid.splits) break;
                const v2f ml_here = both[32 * (s0 + k)];
                const float w = __builtin_amdgcn_exp2f(ml_here[0] - m_all);
                l_all += scaled(ml_here[1], ml_here[0] - m_all);
#pragma unroll
                for (int n = 0; n < DT; n++) out[n] += x[k][n] * w;
            }
        }
        if (threadIdx.x == 0) __hip_atomic_store(grid.arrivals + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);       // ready for the next launch
    }

    // ---- normalise and write ----
    float seen = l_all * 0.0f;
#pragma unroll
    for (int n = 0; n < DT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(out[n][e], 0.0f, seen);
    const uint64_t unfit = __builtin_amdgcn_ballot_w64(live && (!(seen == 0.0f) || l_all == 0.0f));
    if (lane == 0) flags[wave] = (int)((unsigned)unfit | (unsigned)(unfit >> 32));
    __syncthreads();
    unsigned again = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) again |= (unsigned)flags[w];
    again = __builtin_amdgcn_readfirstlane(again);
    if (valid && !((again >> frow) & 1)) {
        const float inv = 1.0f / l_all;
        float *o = a.O + ((int64_t)b * a.Sq + i) * a.ldo + (int64_t)head * a.dk;
#pragma unroll
        for (int n = 0; n < DT; n++) {
            const int col = 32 * n + 8 * wave + 4 * fhalf;
            if (!PAD || col < a.dk) *reinterpret_cast<v4f *>(o + col) = live ? out[n] * inv : v4f{0.f, 0.f, 0.f, 0.f};
        }
        if (a.L && wave == 0 && fhalf == 0) a.L[((int64_t)b * a.H + head) * a.Sq + i] = live ? (m_all + __builtin_amdgcn_logf(l_all)) * LN2 : -INFINITY;
    }
    int nth = 0;
    for (unsigned rest = again; rest; rest &= rest - 1, nth++) {
        const int n = __builtin_ctz(rest);
        if (nth % WAVES == wave) attn_fwd_row(a, b, __builtin_amdgcn_readlane(head, n), __builtin_amdgcn_readlane(i, n), lane);
    }
}

template <int DK, bool PAD>
int launch_few(const AttnArgs &a, FewGrid grid) {
    using G = FewGeom<DK>;
    static bool attr_set = false;
    if (!attr_set) {
        AXHIP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>((k_attn_few<DK, PAD>)), hipFuncAttributeMaxDynamicSharedMemorySize, G::SMEM), "hipFuncSetAttribute");
        attr_set = true;
    }
    const int64_t units = (int64_t)a.B * a.Hkv * grid.row_tiles;
    if (grid.splits > 1) {
        grid.parts = static_cast<float *>(workspace((size_t)units * grid.splits * G::PART * sizeof(float)));
        grid.arrivals = strip_counters((size_t)units);
        if (!grid.parts || !grid.arrivals) return AXHIP_ERR_ALLOC;
    }
    note_kernel(grid.splits > 1 ? "attn_few_ranges" : "attn_few");
    hipLaunchKernelGGL((k_attn_few<DK, PAD>), dim3((unsigned)(units * grid.splits)), dim3(64 * WAVES), G::SMEM, kStream, a, grid);
    return check_launch("attn_fwd");
}

}  // namespace

namespace axhip {

// Whether the few-rows form takes the call, and in how many ranges of keys: until there are two workgroups a CU, or one of heads past 64, which hold a CU alone (us, two -> one: 5 tokens of 2
// sequences over 6000 keys, 16 heads, 8 of keys, of 112 52 -> 34, a token of 8 over 4000, 16, 4 of keys, of 96 44 -> 31), each wave with a tile or more.
// Which form: by what each takes, in us.  Tiles: 128 rows a CU, as long as their keys.  Few rows: a step of 32 rows and 32 keys costs the chip so much (the
// wider heads have one workgroup a CU and twice the work), and every further round of workgroups its start.  Within a few per cent where it is close (us, tiles -> this: 1 token
// of 8 sequences over 1000 keys, 8 heads of 32 25.0 -> 13.4, 4 x 4 of [512, 64] causal 22.5 -> 11.8, 16 queries of 4 heads over 16000 keys, 8 heads of 128 711 -> 94, 4 x 2 x 8 of
// [2048, 32] causal 47 -> 34; the other side 32 of [1024, 96] causal 53 -> 146, 64 of [400, 128] 38 -> 93, 128 of [512, 64] 43 -> 70).  Over 135 random calls it chose
// the slower one 7 times, by 1.8 times at most.  Documents hide much of what tiles would walk, which the host cannot know, and cost them a launch; this form fetches what
// is hidden: it has to be a quarter ahead (42 calls of 2, 7 and 30 documents that it takes by that: 1.34 in the mean, 0.77 to 2.6).
bool attn_fwd_few(const AttnArgs &a, int &rc) {
    const int64_t rows = (int64_t)a.G * a.Sq, cus = cu_count();
    FewGrid grid = {};
    grid.row_tiles = (int)((rows + 31) / 32);
    const int64_t units = (int64_t)a.B * a.Hkv * grid.row_tiles, tiles = ((int64_t)a.Sk + 31) / 32;
    if (units > GRID_MOST / 64) return false;
    int64_t splits = ((a.dk > 64 ? 1 : 2) * cus + units - 1) / units;
    if (splits > (tiles + WAVES - 1) / WAVES) splits = (tiles + WAVES - 1) / WAVES;
    if (splits > SPLITS_MOST) splits = SPLITS_MOST;
    if (splits < 1) splits = 1;
    grid.splits = (int)splits;
    if (rows > 32) {
        const int width = (a.dk + 31) / 32 - 1, pack = a.G > 1 && a.Sq <= 64 ? a.G : 1;
        constexpr double TILE_STEP[] = {0.65, 0.95, 1.5, 1.5}, FEW_STEP[] = {1.1e-3, 1.8e-3, 8e-3, 8e-3};
        const int64_t big = (int64_t)a.B * (a.H / pack) * (((int64_t)pack * a.Sq + 127) / 128);
        const int64_t room = cus * (width < 2 ? 2 : 1), few_rounds = (units * splits + room - 1) / room;
        if (big > cus) return false;                 // (more tiles than CUs never lost to this form)
        const double loaded = (double)big / (double)cus, seen = a.causal && a.Sq == a.Sk ? 0.5 : 1.0;
        const double tile_time = 6.0 + (double)tiles * TILE_STEP[width] * (1.0 + 0.45 * loaded);
        const double few_time = 5.5 + (splits > 1 ? 1.5 : 0.0) + 6.0 * (double)(few_rounds - 1) + (double)(units * tiles) * seen * FEW_STEP[width];
        if (few_time >= (a.doc_k ? 0.75 * (tile_time + 5.0) : tile_time)) return false;
    }
    auto run = [&](auto width) {
        constexpr int DK = decltype(width)::value;
        return a.dk < DK ? launch_few<DK, true>(a, grid) : launch_few<DK, false>(a, grid);
    };
    rc = a.dk <= 32 ? run(std::integral_constant<int, 32>()) : a.dk <= 64 ? run(std::integral_constant<int, 64>()) : a.dk <= 96 ? run(std::integral_constant<int, 96>())
                                                                                                                  : run(std::integral_constant<int, 128>());
    return true;
}

}  // namespace axhip
