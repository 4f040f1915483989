// The form of sxb_attn_decode for many rows (BF16 cache, heads of 128): products on tcgen05, accumulators in tensor memory.  Part of attn_decode.cu.
//
//   S [128 rows, 128 keys] = Q K^T,   P = exp2(S * scale - M),   O [128 rows, 128 columns] += P V
//
// K and V lie in shared memory as they lie in the cache, a line a key; the second product reads V across its lines and P from tensor memory, where P takes
// S's place.  Eight warps make weights: a thread has a row and half of a tile's keys, with a maximum, a sum and sums of values of that half's own, which
// are joined at a segment's end, so that no thread waits for another one's scores.  The maximum that a row goes by is raised, and its sums scaled, only by a
// tile that passes it by more than 2^kSlack.  One warp issues the products, the next tile's scores ahead of this one's weights; three fetch, a stage each.
//
// Measured (B200): 2048 tokens of eight heads a key head on 8192 keys, four key heads, 290 us, 830 TFLOP/s of what the mask leaves; a tile of 128 x 128 takes about
// 2000 cycles, of which the products are 1230 and the exponentials 1024.  64 rows over 64 sequences of 100 to 8000 keys 136 us (bytes alone 81): there a tile
// is half empty, and a sequence's start and end, 5000 cycles, count.  Two warps' scores of one row with one maximum (a barrier of the two a tile) took 497 us
// in the first case, the copies by cp.async (three warps, a third of each tile's rows) 294, boxes of sixteen rows whatever the pages 343.

template <int STAGES> struct TcMisc {
    float top[2][128], sum[2][128];
    int64_t scan[12 + 2];
    uint64_t full[STAGES], values[STAGES], empty[STAGES], scores_done[2], weights[2], sums_done, queries, drained;
    Segment segments[STAGES + 1];       // of what is on its way, and of the tile whose sums go out
    Cursor cur[3];
    uint32_t tmem;
    int abort, how[2];                  // what becomes of a tile's weights: kMma, kMade, kNone
};
constexpr int kMma = 0, kMade = 1, kNone = 2;  // the MMA takes them, the threads have, no row sees the tile
struct TcShape {
    static constexpr int D = 128, BITS = 16, R = 128;
    static constexpr int kSums = 8, kLoads = 3, kStages = kLoads;                  // warps that have the scores and sums, warps that fetch
    static constexpr int kWarps = kSums + kLoads + 1, kThreads = 32 * kWarps, RUN = 16, TK = 128, kPerSm = 1;
    static constexpr int RB = 2 * D, CR = RB / 16;
    static constexpr int kPlane = TK * 128, kTile = 2 * kPlane, kStage = 2 * kTile;  // 64 columns of a tile's keys (lines of 128 bytes); keys or values; both
    static constexpr int kQ = R * D * 2;
    static constexpr int H = TK / 2;                             // keys that a thread has in registers at a time
    static constexpr int kColumns = 512;                         // of tensor memory: scores and weights of two tiles, two halves' sums
    static constexpr int kSmem = kStages * kStage + kQ + (int)sizeof(TcMisc<kStages>);
    static constexpr bool kJoinHere = false;
    static_assert(kSmem <= 227 * 1024, "");
};

// Descriptor of an operand whose rows (or columns) stand side by side in 128-byte lines, a line a k: eights of lines 1024 bytes apart, the next 64 rows
// `plane` bytes on.
__device__ inline uint64_t smem_desc_across(uint32_t addr, uint32_t plane) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(plane >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, BF16 operands, FP32 sums, 128 x 128: bit 16 for a B that lies across.
__device__ constexpr uint32_t tc_instr(bool across) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24) | (across ? 1u << 16 : 0u);
}
__device__ inline void tc_mma_if(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
                 : "memory");
}
// The same with A in tensor memory.
__device__ inline void tc_mma_ts_if(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
                 : "memory");
}
__device__ inline uint32_t tc_ld1(uint32_t at) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(at) : "memory");
    return r;
}
// 32 columns of this thread's lane of tensor memory.
__device__ inline void tc_ld32(uint32_t at, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ inline void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
                 : "memory");
}

// A run of keys of pages of eight tokens or with a bad page: each row looks its page up, rows out of range become zeros, the keys of a bad page NaN.
template <class S>
__device__ __noinline__ void load_rows(const Args &a, const int32_t *table, uint32_t to0, int run0, int lo, int len, int head, int b, int lane) {
    const int page_mask = (1 << a.c.page_shift) - 1, chunk = lane & 15, j0 = run0 + (lane & 15);
    // lane r has the page of row r
    int mine = -1;
    const bool there = j0 >= lo && j0 < len;
    if (there) {
        mine = table[j0 >> a.c.page_shift];
        if ((unsigned)mine >= (unsigned)a.c.n_pages) {
            raise_error(a.err, (uint32_t)b, (uint32_t)mine);
            mine = -2;
        }
    }
#pragma unroll 1
    for (int r0 = 0; r0 < S::RUN; r0 += 2) {
        const int r = r0 + (lane >> 4), id = __shfl_sync(0xffffffffu, mine, r);
        const int64_t off = id < 0 ? 0 : kv_row(a.c, id, head, (run0 + r) & page_mask) * S::RB + chunk * 16;
        const uint32_t to = to0 + (chunk >> 3) * S::kPlane + swz(r, chunk & 7);
        if (id == -2) store_nan<16>(to);
        else copy_async<16>(to, a.c.k + off, id < 0 ? 0 : 16);
        copy_async<16>(to + S::kTile, a.c.v + off, id < 0 ? 0 : 16);
    }
}

// Barriers of the warps that have the sums.
template <class S> __device__ inline void sums_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kSums) : "memory"); }
template <class S> __device__ inline bool sums_any(bool mine) {
    int any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((int)mine), "n"(32 * S::kSums) : "memory");
    return any != 0;
}
// A wait ran out, or the news came that another warp's has: the first one is recorded, and every other wait ends.
__device__ __noinline__ void give_up(const Args &a, int *abort, uint32_t role) {
    if (atomicExch(abort, 1) == 0 && atomicCAS(&a.status[0], 0u, 2u) == 0u) a.status[1] = blockIdx.x, a.status[2] = role;
}
template <class S>
__global__ void __launch_bounds__(S::kThreads, 1) attn_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    constexpr int D = S::D, R = S::R, H = S::H, TK = S::TK, RUN = S::RUN, kStages = S::kStages, kSumThreads = 32 * S::kSums;
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    uint8_t *const q_tile = tc_smem_raw + kStages * S::kStage;
    auto &ms = *reinterpret_cast<TcMisc<kStages> *>(q_tile + S::kQ);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    behind_grid();
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&ms.full[s], 2), mbar_init(&ms.values[s], 2), mbar_init(&ms.empty[s], 1);
        for (int b = 0; b < 2; ++b) mbar_init(&ms.scores_done[b], 1), mbar_init(&ms.weights[b], S::kSums);
        mbar_init(&ms.sums_done, 1), mbar_init(&ms.queries, S::kSums), mbar_init(&ms.drained, 1), ms.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Share share;
    if (!find_share<S>(a, ms.scan, share)) return;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)), "r"(S::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // where the loads begin, and the first segment
    Cursor start;
    start.b = share.b, start.s = sequence<S>(a, start.b), start.segment = 0;
    {
        const int64_t per_head = (int64_t)start.s.tiles * start.s.row_tiles;
        start.head = (int)(share.in / per_head), start.row_tile = (int)((share.in - start.head * per_head) / start.s.tiles);
    }
    auto segment_of = [&](const Cursor &c, int at) { return Segment{c.s.q0, c.s.n, c.s.len, c.s.p0, c.s.lo, c.s.tile0, c.s.tiles, c.head, c.row_tile * R, at, (int)c.s.bad}; };
    if (tid == 32) ms.segments[0] = segment_of(start, (int)(share.in % start.s.tiles));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms.tmem, smem0 = smem_of(tc_smem_raw);
    const int units = (int)(share.u1 - share.u0);
    bool ok = true;
    int last = -1;  // the fill that a copy warp has issued

    if (warp >= S::kSums + 1) {
        // ---- loads: a warp has a stage, and so every third tile ----
        const int stage = warp - S::kSums - 1;
        Cursor &cur = ms.cur[stage];
        if (lane == 0) cur = start;
        __syncwarp();
        const int page_mask = (1 << a.c.page_shift) - 1;
        const uint32_t tile_to = smem0 + stage * S::kStage;
        const int boxes = TK / a.box_rows;
        int at = (int)(share.in % cur.s.tiles), skip = stage;
#pragma unroll 1
        for (int i = stage; i < units; i += kStages, skip = kStages) {
            for (at += skip; at >= cur.s.tiles;) at -= cur.s.tiles, next_segment<S>(a, cur, lane);
            const int32_t *const table = a.pages + cur.b * a.pages_ld;
            const int lo = cur.s.lo, len = cur.s.len, head = cur.head, run0 = (cur.s.tile0 + at) * TK;
            // Lane x has box x, sixteen to 64 keys of a page.  It comes whole where a row may see a key of it, what lies behind the sequence's end in the page too; one
            // that nobody sees does not come: the scores of both are put out of sight and their values' places filled with zeros before the product.
            const int first = run0 + lane * a.box_rows, to = tile_to + lane * (a.box_rows * 128);
            const bool seen = lane < boxes && first < len && first + a.box_rows > lo;
            int page = -1;
            if (seen && page_mask >= 15) page = table[first >> a.c.page_shift];
            const bool fine = (unsigned)page < (unsigned)a.c.n_pages;
            const uint32_t ragged = __ballot_sync(0xffffffffu, seen && !fine), bytes = __popc(__ballot_sync(0xffffffffu, fine)) * (a.box_rows * S::RB);
            if (i >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&ms.empty[stage], (i / kStages - 1) & 1, &ms.abort, a.wait_limit_ns));
            if (!ok) {
                give_up(a, &ms.abort, kRoleAttnCopy);
                break;
            }
            if (blockIdx.x == 0 && i == a.test_skip_slot) continue;  // the test hook's fill never comes
            last = i;
            if (at == 0 && i > 0 && lane == 0) ms.segments[cur.segment % (kStages + 1)] = segment_of(cur, 0);
            if (lane == 0) mbar_expect_tx(&ms.full[stage], bytes), mbar_expect_tx(&ms.values[stage], bytes);
            __syncwarp();
            if (fine) {
                const int row = first & page_mask;
#pragma unroll
                for (int x = 0; x < 2; ++x) tma_load_4d(to + x * S::kPlane, &k_map, 64 * x, row, head, page, &ms.full[stage]);
#pragma unroll
                for (int x = 0; x < 2; ++x) tma_load_4d(to + S::kTile + x * S::kPlane, &v_map, 64 * x, row, head, page, &ms.values[stage]);
            }
            __syncwarp();
            if (SXB_RARE(ragged != 0)) {
#pragma unroll 1
                for (int x = 0; x < TK / RUN; ++x)
                    if ((ragged >> (x * RUN / a.box_rows) & 1) != 0) load_rows<S>(a, table, tile_to + x * (RUN * 128), run0 + x * RUN, lo, len, head, cur.b, lane);
                commit_async();
                wait_async<0>();
                fence_proxy_async();
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&ms.full[stage]), mbar_arrive(&ms.values[stage]);
        }
    } else if (warp == S::kSums) {
        // ---- products ----
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint64_t q_desc = smem_desc(smem_of(q_tile)), k_desc = smem_desc(smem0), v_desc = smem_desc_across(smem0 + S::kTile, S::kPlane);
        int left = 0, segment = 0;  // tiles of the segment behind tile i
        auto wait = [&](uint64_t *bar, int n) {  // for its phase n
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, n & 1, &ms.abort, a.wait_limit_ns));
            if (SXB_RARE(!ok)) give_up(a, &ms.abort, kRoleAttnMma);
            tc_fence_after();
        };
        auto scores = [&](int i) {
            const int stage = i % kStages;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                tc_mma_if(leader, tmem + (i & 1) * TK, q_desc + ((k / 4) * S::kPlane + (k % 4) * 32) / 16, k_desc + (stage * S::kStage + (k / 4) * S::kPlane + (k % 4) * 32) / 16,
                          tc_instr(false), k != 0);
            tc_commit_if(leader, &ms.scores_done[i & 1]);
        };
        bool asked = false, more = false;  // the tile's scores are on their way; there are sums
#pragma unroll 1
        for (int i = 0; i < units && ok; ++i) {
            if (left == 0) {
                wait(&ms.full[i % kStages], i / kStages);
                wait(&ms.queries, segment);
                if (!ok) break;
                const Segment &sg = ms.segments[segment++ % (kStages + 1)];
                left = min(sg.tiles - sg.at, units - i), more = false;
                scores(i);
            } else if (!asked) {
                wait(&ms.full[i % kStages], i / kStages);
                if (!ok) break;
                scores(i);
            }
            --left;
            asked = left > 0 && __all_sync(0xffffffffu, mbar_test(&ms.full[(i + 1) % kStages], ((i + 1) / kStages) & 1));
            if (asked) {
                tc_fence_after();
                scores(i + 1);
            }
            wait(&ms.weights[i & 1], i >> 1);
            wait(&ms.values[i % kStages], i / kStages);
            if (!ok) break;
            const int stage = i % kStages, how = ms.how[i & 1];
            if (how == kMma) {
#pragma unroll
                for (int k = 0; k < TK / 16; ++k)
                    tc_mma_ts_if(leader, tmem + 2 * TK + (k / 4) * D, tmem + (i & 1) * TK + (k / 4) * H + (k % 4) * 8, v_desc + (stage * S::kStage + k * 2048) / 16, tc_instr(true), more || k % 4 != 0);
            }
            more = more || how != kNone;
            tc_commit_if(leader, &ms.empty[stage]);
            tc_commit_if(leader, &ms.sums_done);
        }
    } else {
        // ---- scores and sums ----
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes_at = tmem + ((uint32_t)(warp & 3) << 21), sums_at = lanes_at + 2 * TK + half * D;
        auto wait = [&](uint64_t *bar, int n) {  // for its phase n
            ok = ok && mbar_wait(bar, n & 1, &ms.abort, a.wait_limit_ns);
            if (SXB_RARE(!ok)) give_up(a, &ms.abort, kRoleAttnSums);
            __syncwarp();
            tc_fence_after();
        };
        // what this warp had of tensor and shared memory is read, or written
        auto tell = [&](uint64_t *bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        const float fac = a.softcap > 0.f ? 1.f : a.scale * kLog2e;
        int segment = 0;

#pragma unroll 1
        for (int first = 0, n; first < units; first += n, ++segment) {
            const Segment &sg = ms.segments[segment % (kStages + 1)];
            if (first > 0) {  // (the record comes with its first tile, the first one's has been there)
                wait(&ms.full[first % kStages], first / kStages);
                if (sums_any<S>(!ok)) break;
            }
            n = min(sg.tiles - sg.at, units - first);
            const int rows = min(R, sg.n * a.group - sg.rows0), tok = (sg.rows0 + row) / a.group, head = sg.head * a.group + sg.rows0 + row - tok * a.group;
            {   // the segment's queries: a thread half a row
                uint4 w[8] = {};
                if (row < rows) {
                    const auto *const from = reinterpret_cast<const uint4 *>(a.q + (sg.q0 + tok) * a.q_ld + (int64_t)head * D + half * 64);
#pragma unroll
                    for (int c = 0; c < 8; ++c) w[c] = from[c];
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4 *>(q_tile + half * S::kPlane + swz(row, c)) = w[c];
            }
            fence_proxy_async();
            tell(&ms.queries);
            // what the row sees, and the tiles that all of them see all of
            const int hi = row < rows ? sg.p0 + tok : -1, lo = a.window > 0 ? (int)max((int64_t)-1, (int64_t)hi - a.window) : -1;
            const int hi0 = sg.p0 + sg.rows0 / a.group, hi1 = sg.p0 + min(sg.n - 1, (sg.rows0 + R - 1) / a.group), from = a.window > 0 ? max(0, hi1 - a.window + 1) : 0;
            const int whole0 = (from + TK - 1) / TK, whole1 = (hi0 + 1 + TK) / TK - 1, lo0 = a.window > 0 ? (int)max((int64_t)-1, (int64_t)hi0 - a.window) : -1;
            const bool idle = (warp & 3) * 32 >= rows;  // no row of the warp is one: what stands in its lanes nobody reads
            float top = kLowest, l = 0.f;
            bool more = false;

#pragma unroll 1
            for (int i = first; i < first + n; ++i) {
                const int tile = sg.tile0 + sg.at + i - first, j0 = tile * TK + half * H;
                const bool whole = tile >= whole0 && tile < whole1;
                const uint32_t scores_at = lanes_at + (i & 1) * TK + half * H;
                int how = kMma;
                wait(&ms.scores_done[i & 1], i >> 1);
                if (SXB_RARE(!whole) && (tile * TK > hi1 || tile * TK + TK - 1 <= lo0)) {
                    how = kNone;
                } else if (!idle) {
                    uint4 w[H / 8];
                    float sum;
#pragma unroll 1
                    for (int pass = 0; pass < 2; ++pass) {
                        float most = -CUDART_INF_F;
                        uint64_t sums = pair(0.f, 0.f);
                        float s[H];
#pragma unroll
                        for (int c = 0; c < H; c += 32) tc_ld32(scores_at + c, s + c);
                        if (SXB_RARE(a.softcap > 0.f)) {
                            const float by = 2.f / a.softcap, to = a.softcap * kLog2e;
#pragma unroll
                            for (int c = 0; c < H; ++c) s[c] = capped(s[c], a.scale * kLog2e, by, to);
                        }
                        if (SXB_RARE(!whole)) {
                            const int above = hi - j0, below = lo - j0;
#pragma unroll
                            for (int c = 0; c < H; ++c)
                                if (c > above || c <= below) s[c] = -CUDART_INF_F;
                        }
                        const uint64_t fac2 = pair(fac, fac), top2 = pair(-top, -top);
#pragma unroll
                        for (int c = 0; c < H; c += 2) {
                            most = fmaxf(most, fmaxf(s[c], s[c + 1]));
                            float x0, x1;
                            unpair(fma_pair(pair(s[c], s[c + 1]), fac2, top2), x0, x1);
                            const float p0 = exp2_flushed(x0), p1 = exp2_flushed(x1);
                            sums = add_pair(pair(p0, p1), sums);
                            reinterpret_cast<uint32_t *>(w)[c / 2] = pack_bf16(p0, p1);
                        }
                        float odd;
                        unpair(sums, sum, odd);
                        sum += odd;
                        most *= fac;
                        if (pass == 1 || !SXB_RARE(__any_sync(0xffffffffu, most - top > (float)kSlack))) break;
                        // the row's maximum from here on, and what there is of its sums
                        const float now = fmaxf(top, most), f = exp2_flushed(top - now);
                        top = now, l *= f;
                        if (more) {
                            wait(&ms.sums_done, i - 1);
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                float o[16];
                                uint4 d[4];
                                tc_ld16(sums_at + c, o);
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    d[x] = make_uint4(__float_as_uint(o[4 * x] * f), __float_as_uint(o[4 * x + 1] * f), __float_as_uint(o[4 * x + 2] * f), __float_as_uint(o[4 * x + 3] * f));
                                tc_st16(sums_at + c, d);
                            }
                        }
                    }
                    l += sum;
#pragma unroll
                    for (int c = 0; c < H / 32; ++c) {
                        const uint4 d[4] = {w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
                        tc_st16(scores_at + 16 * c, d);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                // Values of keys that no row sees become zeros, whatever they are: 0 * v has to be 0.  Of keys that one row sees and another does not, an infinity or a
                // NaN must not reach the other: the threads add such a tile's up, each for its row.
                if (SXB_RARE(!whole && how == kMma)) {
                    bool odd = false;
                    wait(&ms.values[i % kStages], i / kStages);
                    uint8_t *const vt = tc_smem_raw + (i % kStages) * S::kStage + S::kTile;
#pragma unroll 1
                    for (int c = tid; c < S::kTile / 16; c += kSumThreads) {
                        auto *const at = reinterpret_cast<uint4 *>(vt + c * 16);
                        const int j = tile * TK + (c >> 3) % TK;
                        if (j > hi1 || j <= lo0) {
                            *at = make_uint4(0, 0, 0, 0);
                        } else if (sg.n > 1) {
                            const uint4 v = *at;
                            const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) odd = odd || (vs[e] & 0x7f80u) == 0x7f80u || (vs[e] & 0x7f800000u) == 0x7f800000u;
                        }
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (SXB_RARE(sums_any<S>(odd))) {
                        how = kMade;
                        if (!idle) {
                            if (more) wait(&ms.sums_done, i - 1);
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                float o[16];
                                if (more) {
                                    tc_ld16(sums_at + c, o);
                                } else {
#pragma unroll
                                    for (int x = 0; x < 16; ++x) o[x] = 0.f;
                                }
#pragma unroll 1
                                for (int k = 0; k < H; ++k) {
                                    const uint32_t p2 = tc_ld1(scores_at + k / 2);
                                    const float p = __uint_as_float(k & 1 ? p2 & 0xffff0000u : p2 << 16);
                                    if (j0 + k <= hi && j0 + k > lo) {
#pragma unroll
                                        for (int x = 0; x < 16; ++x)
                                            o[x] = fmaf(p, bf16_bits_to_f32(*reinterpret_cast<const uint16_t *>(vt + (c >> 6) * S::kPlane + swz(half * H + k, ((c & 63) + x) >> 3) + (x & 7) * 2)), o[x]);
                                    }
                                    __syncwarp();
                                }
                                uint4 d[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x) d[x] = make_uint4(__float_as_uint(o[4 * x]), __float_as_uint(o[4 * x + 1]), __float_as_uint(o[4 * x + 2]), __float_as_uint(o[4 * x + 3]));
                                tc_st16(sums_at + c, d);
                            }
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        }
                    }
                }
                if (tid == 0) ms.how[i & 1] = how;
                tell(&ms.weights[i & 1]);
                more = more || how != kNone;
                if (SXB_RARE((i & 63) == 63) && sums_any<S>(!ok)) break;  // no tile after tile of a segment that nobody finishes
            }

            // ---- the segment's end, or this CTA's share's: the halves' sums, each by what its maximum is below the higher one ----
            const int64_t seg0 = share.u0 + first - sg.at, seg1 = seg0 + sg.tiles;
            const bool split = seg0 < share.u0 || seg1 > share.u1;
            ms.top[half][row] = top, ms.sum[half][row] = l;
            wait(&ms.sums_done, first + n - 1);
            if (sums_any<S>(!ok)) break;
            tc_fence_after();
            const float top0 = ms.top[0][row], top1 = ms.top[1][row], both = fmaxf(top0, top1);
            float f0 = exp2_flushed(top0 - both), f1 = exp2_flushed(top1 - both);
            const float all = fmaf(ms.sum[0][row], f0, ms.sum[1][row] * f1), inv = split ? 1.f : sg.bad ? qnan_f32() : all == 0.f ? 0.f : 1.f / all;
            f0 *= inv, f1 *= inv;
            float *const part = a.partial + (2 * (int64_t)blockIdx.x + (seg0 < share.u0 ? 0 : 1)) * R * (D + 2);
            if (half == 0 && row < rows) {
                if (split) part[R * D + row] = both, part[R * (D + 1) + row] = all;
                else if (a.lse != nullptr) a.lse[(int64_t)(sg.q0 + tok) * a.n_q + head] = sg.bad ? qnan_f32() : all == 0.f ? -CUDART_INF_F : fmaf(both, kLn2, logf(all));
            }
            if (split && tid == 0 && seg0 >= share.u0) {
                auto cta_of = [&](int64_t u) { return ((u + 1) * share.ctas + share.total - 1) / share.total - 1; };
                a.joins[blockIdx.x] = Join{sg.q0, sg.rows0, sg.head, rows, (int)(cta_of(seg1 - 1) - cta_of(seg0)) + 1, {}};
            }
            if (!idle) {
#pragma unroll 1
                for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 16) {
                    float o0[16], o1[16];
                    tc_ld16x2(lanes_at + 2 * TK + c, lanes_at + 2 * TK + D + c, o0, o1);
#pragma unroll
                    for (int x = 0; x < 16; ++x) o0[x] = more ? fmaf(o0[x], f0, o1[x] * f1) : 0.f * inv;
                    if (row < rows) {
                        if (split) {
                            auto *const to = reinterpret_cast<float4 *>(part + row * D + c);
#pragma unroll
                            for (int x = 0; x < 4; ++x) to[x] = make_float4(o0[4 * x], o0[4 * x + 1], o0[4 * x + 2], o0[4 * x + 3]);
                        } else {
                            auto *const to = reinterpret_cast<uint4 *>(a.out + (sg.q0 + tok) * a.out_ld + (int64_t)head * D + c);
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                to[x] = make_uint4(pack_bf16(o0[8 * x], o0[8 * x + 1]), pack_bf16(o0[8 * x + 2], o0[8 * x + 3]), pack_bf16(o0[8 * x + 4], o0[8 * x + 5]),
                                                   pack_bf16(o0[8 * x + 6], o0[8 * x + 7]));
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            sums_sync<S>();
        }
        // A CTA that has given up has parts that others' are joined with, of an earlier call: their sums of weights become NaN, and so do the rows.
        if (*static_cast<volatile int *>(&ms.abort) != 0 && half == 0) {
            float *const sums = a.partial + 2 * (int64_t)blockIdx.x * R * (D + 2) + R * (D + 1) + row;
            if (segment == 0) sums[0] = qnan_f32();
            sums[R * (D + 2)] = qnan_f32();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (SXB_RARE(*static_cast<volatile int *>(&ms.abort) != 0)) {
        // Nothing may still be on its way when shared and tensor memory go to another CTA: each copy warp waits for its last fill, the MMA warp for its products.
        if (warp > S::kSums && last >= 0) {
            const int stage = warp - S::kSums - 1;
            mbar_wait(&ms.full[stage], (last / kStages) & 1, nullptr, 1000000ull), mbar_wait(&ms.values[stage], (last / kStages) & 1, nullptr, 1000000ull);
        } else if (warp == S::kSums) {
            tc_commit_if(elect_one() ? 1u : 0u, &ms.drained);
            mbar_wait(&ms.drained, 0, nullptr, 1000000ull);
        }
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
    }
}
