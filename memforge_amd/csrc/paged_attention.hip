// Planners and C entry points of the varlen paged attention (the kernels are in
// attn_kernels.h).
#include <atomic>
#include <exception>
#include <mutex>
#include <vector>

#include "attn_kernels.h"

namespace {
// The planner of mf_attention_plan (num_cus 0), mf_attention_plan_device,
// mf_attention_plan_merge_free (cut false) and mf_attention_plan4 (four).
int attention_plan(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens, int num_q_heads,
                   int num_kv_heads, int head_dim, int dtype, int partition_tiles, int num_cus, bool cut, int32_t* items,
                   int64_t items_capacity, int32_t* merges, int64_t merges_capacity, int64_t* counts,
                   bool four = false) {
    if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || !counts)
        return MF_ERR_ARG;
    if (num_q_heads % num_kv_heads) return MF_ERR_ARG;
    if (num_seqs > 0 && (!cu_seqlens || !kv_lens)) return MF_ERR_ARG;
    const int DP = mf::padded_head_dim(dtype, head_dim);
    if (!mf::dtype_ok(dtype) || !DP) return MF_ERR_UNSUPPORTED;
    const int WT = mf::wide_tiles(dtype, DP);
    const int G = num_q_heads / num_kv_heads;
    const int Hkv = num_kv_heads;

    auto col_tiles = [&](int s) -> int {
        const int qlen = cu_seqlens[s + 1] - cu_seqlens[s];
        if (qlen <= 0 || kv_lens[s] <= 0) return 0;
        return (qlen * G + 15) / 16;
    };

    // Key partition sizes, per item class. Single-column-tile (narrow)
    // items get their parallelism from splitting keys: about MF_NARROW_ITEMS
    // items (two to four waves per SIMD), few enough that partials stay
    // small. (Measured on C5: 128-tile partitions, 4,192 items, beat 64-tile
    // ones, 7,320 items: 539 vs 548 us and a merge of 13.5 vs 20 us.) Wide items already
    // come as many column groups, and each split of one costs a 16-column fp32
    // partial per tile written and merged again, so they are split only as far
    // as it takes to reach kWideItems items.
    // Narrow partition: the candidate (a power of two from 4 to
    // kMaxItemTiles tiles per wave) with the least estimated time, where a
    // launch takes the longer of its bandwidth time and its longest wave's
    // chain of tiles, plus the merge launch if any range is split. A range of
    // T > q tiles runs as ceil(T / 4q) units of four waves. Ties go to the
    // longer partition. The constants are fitted to partition sweeps on
    // MI355X (bf16, D 64) timed as HIP-graph replays, i.e. without host
    // submission time: a lone wave's chain costs about 0.53 us per 16-key
    // tile, decode items stream near 5 TB/s, and a split costs about 9 us of
    // merge. Picks: merge-free 32-tile waves for a 64-sequence decode step of
    // 96-1152 keys (17.0 us against 18.5 at 4 tiles), 8 for C3's verify (16.8
    // against 18.5 merge-free at 32), 16 for C2's decodes, 128 on C5.
    auto narrow_partition = [&](int fallback) {
        constexpr double kChainUs = 0.53, kMergeUs = 9.0, kBytesPerUs = 5.0e6;
        const double tile_us = 16.0 * DP * mf::dtype_size(dtype) * 2 / kBytesPerUs;
        int64_t tiles_all = 0;
        for (int s = 0; s < num_seqs; ++s) {
            const int nct = col_tiles(s);
            if (nct && (nct == 1 || WT == 1)) tiles_all += (int64_t)Hkv * nct * ((kv_lens[s] + 15) / 16);
        }
        if (!tiles_all) return fallback;
        int best_q = fallback;
        double best = 1e300;
        for (int q = 4; q <= mf::kMaxItemTiles; q *= 2) {
            int longest = 0;
            bool split = false;
            for (int s = 0; s < num_seqs; ++s) {
                const int nct = col_tiles(s);
                if (!nct || !(nct == 1 || WT == 1)) continue;
                const int T = (kv_lens[s] + 15) / 16;
                if (T <= q) {
                    longest = std::max(longest, T);
                    continue;
                }
                const int units = (T + 4 * q - 1) / (4 * q);
                const int unit = (T + units - 1) / units;
                longest = std::max(longest, (unit + 3) / 4);
                split = split || units > 1;
            }
            const double est = std::max(tiles_all * tile_us, longest * kChainUs) + (split ? kMergeUs : 0.0);
            if (est <= best) {
                best = est;
                best_q = q;
            }
        }
        return best_q;
    };
    int64_t work = 0, wide_units = 0, narrow_units = 0;
    int wide_max_tiles = 0;
    for (int s = 0; s < num_seqs; ++s) {
        const int nct = col_tiles(s);
        if (!nct) continue;
        const bool narrow = nct == 1 || WT == 1;
        const int groups = narrow ? nct : (nct + WT - 1) / WT;
        const int tiles = (kv_lens[s] + 15) / 16;
        work += (int64_t)Hkv * groups * tiles;
        if (narrow) narrow_units += (int64_t)Hkv * groups;
        if (!narrow) {
            wide_units += (int64_t)Hkv * groups;
            wide_max_tiles = std::max(wide_max_tiles, tiles);
        }
    }
    int P = std::min(partition_tiles, mf::kMaxItemTiles);
    int PW = P;
    bool mixed = false;  // a shared launch of narrow and wide items (quad partitions below)
    if (P <= 0) {
        const int64_t target_items = MF_NARROW_ITEMS;
        int64_t want = (work + target_items - 1) / target_items;
        int PA = 4;
        while (PA < want && PA < mf::kMaxItemTiles) PA *= 2;
        P = narrow_partition(PA);
        // wide: the smallest partition (a power of two, at least PA) whose
        // item count stays within the target
        PW = PA;
        if (wide_units > 0) {
            auto wide_items = [&](int q) {
                int64_t n = 0;
                for (int s = 0; s < num_seqs; ++s) {
                    const int nct = col_tiles(s);
                    if (!nct || nct == 1 || WT == 1) continue;
                    n += (int64_t)Hkv * ((nct + WT - 1) / WT) * (((kv_lens[s] + 15) / 16 + q - 1) / q);
                }
                return n;
            };
            while (PW < mf::kMaxItemTiles && PW < wide_max_tiles && wide_items(PW) > MF_WIDE_ITEMS) PW *= 2;
            // Beside wide items the narrow ones run in the same launch
            // (attn_mixed_kernel), where a narrow chain as long as a wide
            // wave's key range is hidden behind the wide waves; longer
            // narrow partitions then only save items and merges. Measured
            // on the C2 step (PW 32): narrow P 16 (the estimate's pick)
            // 58.1-58.9 us per layer, P 32 56.6-56.8, P 64 60.3-60.5;
            // again with the KV write in the launch and the raised prefill
            // priority: P 16 57.0-57.3, P 32 48.9-49.3, P 64 58.1-58.3.
            // The planner does not see the pool's block size: the shared
            // launch needs 16-key blocks, and with other block sizes the two
            // classes run as separate launches, where the raised partition
            // only lengthens the narrow launch's chains (no effect on
            // results, which do not depend on the partition).
            if (MF_MIXED_LAUNCH && WT > 1 && dtype != MF_F32 && head_dim == DP && narrow_units > 0) {
                P = std::max(P, PW);
                mixed = true;
            }
        }
    }

    // Narrow items (one 16-column tile): a (sequence, kv head, column tile)
    // of at most P key tiles is one single-wave item, packed four to a
    // workgroup with other single items. A longer one is cut into balanced
    // units of at most 4P tiles; a unit is a cooperative workgroup whose four
    // waves take consecutive quarters of its tiles and combine their softmax
    // states through LDS, so only ranges of more than 4P tiles leave split-K
    // partials for the merge kernel.
    //
    // Wide items are launched in workgroups of kWaves (one item per wave).
    // A (sequence, kv head, partition) run of at least kWaves column groups
    // fills whole workgroups of its own -- consecutive column groups, the last
    // one padded with empty items (no column tiles) -- so the workgroup shares
    // each K/V tile through LDS. Shorter runs are pooled and packed kWaves to
    // a workgroup, each wave on its own keys.
    const int U = mf::kWaves;
    // Decode steps planned for a device (one row a sequence, one column tile
    // each) that the general partition leaves with fewer than two workgroups
    // per compute unit. Where its longest chain of tiles sets the time,
    // ranges run as cooperative units from a few tiles on: above 4 / 16 / 32
    // tiles with up to one / two / more (sequence, kv head) pairs per compute
    // unit, and always above P, the most a single wave of the general partition
    // takes (a longer range left to one wave would also lose its tiles past P;
    // us as four-wave units, then as single waves: 64 sequences of 256 keys at
    // 15/5 heads x 64 6.4, 8.5; 40 of 256 at 40/8 x 128 12.8, 17.9; 120 of up to
    // 256 at 9/3 x 64 5.1, 8.1). At 256-byte rows a range is cut where the
    // longest holds more than 80 tiles into units of
    // about total / (1.8 x compute units) tiles, at least 32 and at most 72: two
    // workgroups of a unit per compute unit and one round of them. At 128-byte
    // rows, whose tiles chain three times as fast, a step with ranges of more
    // than 100 tiles keeps the general plan, which cuts those well (59 sequences
    // of up to 2800 keys at 9/3 x 64 19.6 us against 22.7 cut as above).
    // Measured, us, general plan then this one: 64 sequences of up to 1152 keys
    // at 15/5 x 64 17.4, 15.3 (units of 64 tiles and merges 19.2); at 40/8 x 128
    // 4 of 8192 to 24576 84, 66 (units of 128 tiles 76, 256 84); 16 of 500 to
    // 4000 73, 45 (uncut 71); 64 of 200 to 3000 119, 70 (uncut 85).
    //
    // Which plan takes less time is estimated from the longest chain one wave
    // runs (a tile takes 0.33 us at 4 KB of K and V, 0.95 at 8 KB and in
    // proportion above), the bytes at 5.5 TB/s, and a merge launch of 4 us. Where
    // the bytes set the general plan's time and the two come out about the same,
    // the general plan is kept if its workgroups fill the compute units evenly
    // (its tiles are at least 0.7 of those that every unit's longest would make);
    // else its last workgroups run on a part-empty chip. Graph replays over pools
    // larger than the caches, us, general plan then this one whatever the
    // estimate: 1 sequence of 1400 keys at 9/3 x 64 8.7, 11.0; 4 of 1400 at 15/5
    // x 64 8.9, 11.0; 2 of about 2000 at 40/8 x 128 13.6, 16.8; 100 of 1400 there
    // 105, 128 (even), 33 of 5000 202, 128 (264 workgroups on 256 units). Over
    // 772 steps of 1 to 200 sequences at seven shapes the choice takes 0.1% more
    // than the better plan on average, and 8 take over 5% more.
    int single_max = P;
    double unit_tiles = 0;  // tiles per unit of a cut range (0: the general partition)
    const auto decode_units = [](int tiles, double per_unit) {
        const int n = std::max(1, (int)std::lround(tiles / per_unit));
        return std::max(n, (tiles + mf::kWaves * mf::kMaxItemTiles - 1) / (mf::kWaves * mf::kMaxItemTiles));
    };
    if (four && partition_tiles <= 0 && !mixed) {
        // A 4-bit pool's tile is a quarter of the bytes and about a third of the chain
        // (0.3 us a wave at head_dim 128). Ranges are cut into units for two workgroups
        // a compute unit in all, three below head_dim 128, of at least 64 tiles and at
        // least a 32nd of the longest range (a merge reads its partitions four by four,
        // dealt to four waves), at most 512. Measured, us, at units of 64 / 96 / 160 /
        // 256 / 512 tiles: 4 sequences of 16384 to 65536 keys at 40/8 heads x 128
        // (rule 164) 48 / 46 / 41 / 48 / 54, with the 16-bit rule 56; one of 65536
        // (128) 24.6 / 26 / 21.8 / 25 / 41; 64 of 200 to 3000 (100) 29 / 32 / 27 / 28 /
        // 42; 256 of a median of 2048 (512) 214 / 200 / 190 / 184.5 / 183.4; at 15/5 x
        // 64 32 of 1000 to 8000 (64) 18.5 / 19.4 / 21.8 / 26 / 40.
        int64_t pairs = 0, tiles_all = 0;
        int longest = 0;
        for (int s = 0; s < num_seqs; ++s) {
            const int nct = col_tiles(s);
            if (!nct || !(nct == 1 || WT == 1)) continue;
            const int T = (kv_lens[s] + 15) / 16;
            pairs += (int64_t)Hkv * nct;
            tiles_all += (int64_t)Hkv * nct * T;
            longest = std::max(longest, T);
        }
        const double wgs = (head_dim >= 128 ? 2.0 : 3.0) * num_cus;
        single_max = std::min(P, pairs <= num_cus ? 4 : pairs <= 2 * (int64_t)num_cus ? 16
                                 : pairs <= 4 * (int64_t)num_cus ? 32 : mf::kMaxItemTiles);
        // a few workgroups over a whole round would run alone after it, so the units
        // grow until they fit (32 of 1000 to 8000 at 40/8 x 128: 552 workgroups 42 us,
        // 480 37)
        auto workgroups = [&]() {
            double n = 0;
            for (int s = 0; s < num_seqs; ++s) {
                const int nct = col_tiles(s), T = (kv_lens[s] + 15) / 16;
                if (!nct || !(nct == 1 || WT == 1)) continue;
                n += (double)Hkv * nct * (T <= single_max ? 0.25 : decode_units(T, unit_tiles));
            }
            return n;
        };
        unit_tiles = std::max({64.0, longest / 32.0, tiles_all / wgs});
        while (unit_tiles < 512 && workgroups() > wgs) unit_tiles *= 1.04;
        unit_tiles = std::min(unit_tiles, 512.0);
    } else if (num_cus > 0 && partition_tiles <= 0 && !mixed) {
        int64_t pairs = 0, tiles_all = 0, singles = 0, units = 0;
        int longest = 0;
        bool decode = true;
        for (int s = 0; s < num_seqs; ++s) {
            const int nct = col_tiles(s);
            if (!nct) continue;
            decode = decode && nct == 1 && cu_seqlens[s + 1] - cu_seqlens[s] == 1;
            const int T = (kv_lens[s] + 15) / 16;
            pairs += Hkv;
            tiles_all += (int64_t)Hkv * T;
            longest = std::max(longest, T);
            if (T > P) units += (int64_t)Hkv * ((T + U * P - 1) / (U * P));
            else singles += Hkv;
        }
        const int row_bytes = DP * mf::dtype_size(dtype);
        const bool long_rows = row_bytes >= 256;
        if (decode && units + singles / U < 2 * (int64_t)num_cus && (long_rows || longest <= 100)) {
            const int single = std::min(P, pairs <= num_cus ? 4 : pairs <= 2 * (int64_t)num_cus ? 16 : 32);
            const double per_unit = cut && long_rows && longest > 80
                                        ? std::min(72.0, std::max(32.0, (double)tiles_all / (1.8 * num_cus)))
                                        : 1e9;
            const double tile_us = row_bytes >= 256 ? 0.95 * row_bytes / 256 : 0.33;
            const double bytes_us = (double)tiles_all * 32 * row_bytes / 5.5e6;
            struct Shape {
                double chain_us, us;  // the longest chain's time, the estimate
                double fill;          // tiles over those of a grid of longest workgroups
                bool split;
            };
            auto shape = [&](int alone, auto units_of) {
                int chain = 0, work = 0;
                int64_t waves = 0;
                bool split = false;
                for (int s = 0; s < num_seqs; ++s) {
                    if (!col_tiles(s)) continue;
                    const int T = (kv_lens[s] + 15) / 16;
                    const int n = T <= alone ? 1 : units_of(T);
                    const int unit = (T + n - 1) / n;
                    chain = std::max(chain, T <= alone ? T : (unit + U - 1) / U);
                    work = std::max(work, T <= alone ? U * T : unit);
                    waves += (int64_t)Hkv * (T <= alone ? 1 : U * n);
                    split = split || n > 1;
                }
                const int64_t grid = ((waves + U - 1) / U + num_cus - 1) / num_cus * num_cus;
                return Shape{chain * tile_us, std::max(bytes_us, chain * tile_us) + (split ? 4.0 : 0.0),
                             (double)tiles_all / ((double)grid * std::max(work, 1)), split};
            };
            Shape general = shape(P, [&](int T) { return (T + U * P - 1) / (U * P); });
            if (!cut && general.split) {
                // the plan a merge-free launch gets without the rule: the smallest
                // partition whose units hold the longest range whole
                int q = 4;
                while (U * q < longest && q < mf::kMaxItemTiles) q *= 2;
                general = shape(q, [&](int T) { return (T + U * q - 1) / (U * q); });
            }
            const Shape units_only = shape(single, [&](int T) { return decode_units(T, per_unit); });
            if (units_only.us < 0.995 * general.us ||
                (units_only.us <= 1.2 * general.us && bytes_us >= 0.9 * general.chain_us && general.fill < 0.7)) {
                single_max = single;
                unit_tiles = per_unit;
            }
        }
    }
    auto round_up = [&](int64_t n) { return (n + U - 1) / U * U; };
    // key partitions of sequence s: count, and the start of partition p
    // (narrow cooperative ranges are balanced; the rest are Q-tile strides).
    // A wide range takes as many partitions as PW-tile strides would give,
    // in strides of equal length: the C2 chunks planned prefill-only
    // 34.9-35.3 us against 36.3-36.6 with PW strides (a short last
    // partition).
    auto partitions = [&](int s, bool narrow, int& Q, bool& coop) {
        const int tiles = (kv_lens[s] + 15) / 16;
        coop = narrow && tiles > single_max;
        Q = narrow ? (coop ? U * P : P) : PW;
        if (narrow && unit_tiles > 0) return coop ? decode_units(tiles, unit_tiles) : 1;
        if (!narrow && tiles > PW) {
            const int np = (tiles + PW - 1) / PW;
            Q = (tiles + np - 1) / np;
        }
        return (tiles + Q - 1) / Q;
    };
    auto part_begin = [&](int tiles, int nparts, int Q, bool coop, int p) {
        return coop ? (int)((int64_t)p * tiles / nparts) : std::min(tiles, p * Q);
    };
    // Quad partitions (mixed plans). A sequence whose wide items fill whole
    // workgroups runs as column quads: the kWaves column groups one
    // workgroup holds, over one key range. In a mixed plan each quad takes
    // its own partitions: the tiles its last column sees, cut into
    // round(visible / W) equal ranges, W chosen so that the launch's wide
    // workgroups carry about two rounds' worth per compute unit (the total
    // visible work over 2 x 256 CUs, at least PW). Every wide workgroup then
    // holds about the same work, and each compute unit about two of them
    // beside the narrow ones, all in one resident round. C2 step, engine
    // layer as graph replays: 44.1-44.2 us against 45.8-46.0 with the ranges'
    // partitions (PW 64 strides); 1.5 workgroups per CU 49.3-49.6, 2.5
    // 47.1-47.4, 3 47.5-48.0, 4 53.3-53.5. Plans of wide items only, made without
    // a device, keep the ranges' partitions (there two per CU took the prefill
    // items of the 16x16 loop from 35.1 to 37.9 us). The XCD queues below take a (sequence, kv head)'s quads
    // as one run: the launch fetches 1.09x its algorithmic reads, against
    // 1.65x with each (quad, kv head) dealt alone (0.3 us faster).
    const int kPlanCUs = num_cus > 0 ? num_cus : 256;  // an MI355X has 256 compute units
    // A plan made for a device cuts every wide sequence by quads -- also one of
    // fewer than four column groups, whose quad has idle waves but whose tiles
    // are shared -- and a shared workgroup's range may be any length (its block
    // table is read 64 tiles at a time). At 128-byte rows and less, a plan of
    // wide items only does so where the general ranges come out shorter than 32
    // tiles (PW), and a workgroup's set-up costs more than its tiles: 15/5 heads
    // x 64, device against general ranges, us: 1024 fresh rows (8 tiles) 18.1
    // against 23.9, 8 prompts of up to 300 (4) 14.2 / 18.9, 256 rows after 6144
    // keys (19) 24.3 / 27.7, but 4 chunks of 512 after up to 2048 (32) 25.6 /
    // 28.6 and 16 prompts of up to 1024 (64) 30 / 32. At 256-byte rows it always
    // does: 2 chunks of 2048 after 6144 keys 370 against 428 (10,240 merges).
    const bool device = num_cus > 0 && partition_tiles <= 0 && WT > 1 && dtype != MF_F32 && head_dim == DP &&
                        (mixed || DP >= 128 || PW < 32 || four);
    auto quads = [&](int s) -> int {  // column quads of s, 0 if s is not a shared wide sequence
        const int nct = col_tiles(s);
        if (!(mixed || device) || !nct || nct == 1 || WT == 1) return 0;
        const int ngroups = (nct + WT - 1) / WT;
        return device || ngroups >= U ? (int)(round_up(ngroups) / U) : 0;
    };
    auto quad_visible = [&](int s, int qd) -> int {
        const int rows = cu_seqlens[s + 1] - cu_seqlens[s];
        const int end_ct = std::min(col_tiles(s), (qd + 1) * U * WT);
        const int last_col = std::min(end_ct * 16, rows * G) - 1;
        const int last_pos = kv_lens[s] - rows + last_col / G;
        return std::max(1, std::min((kv_lens[s] + 15) / 16, last_pos / 16 + 1));
    };
    double quad_w = 1.0;
    const int max_range = device ? INT_MAX : mf::kMaxItemTiles;
    if (mixed || device) {
        int64_t visible = 0, quad_units = 0;
        int longest = 0;
        for (int s = 0; s < num_seqs; ++s)
            for (int qd = 0, nq = quads(s); qd < nq; ++qd) {
                const int v = quad_visible(s, qd);
                visible += (int64_t)Hkv * v;
                quad_units += Hkv;
                longest = std::max(longest, v);
            }
        quad_w = std::max((double)std::max(PW, 1), (double)visible / (2.0 * kPlanCUs));
        if (device && !mixed) {
            // About two workgroups per compute unit, of at least 16 tiles (12 at
            // head_dim 128: 7-row verifies of up to 600 keys at 40/8 18.5 us
            // against 21.8 at 16); where that makes ranges longer than 96 tiles, about four, of at
            // least 96. Measured, us at 8 / 16 / 24 / 32 / 48 / 64 / 128 tiles
            // per range and uncut: one chunk of 256 rows after 6144 keys, 15/5
            // heads x 64 33.6 / 27.3 / 24.3 / 24.0 / 24.7 / 29.2 / 38 / 88 (rule
            // 23), 40/8 x 128 99 / 71 / 62 / 66 / 51 / 58 / 79 / 202 (64); 1024
            // fresh rows, x 64 19.8 / 18.1 / 19.1 / 21.4 / 21.0 uncut (16), x 128
            // 50 / 36 / 36 / 41 / 45 uncut (20); 2 chunks of about 850 rows
            // after 4000 keys x 128 714 / 449 / 374 / 335 / 301 / 291 / 295 / 292
            // (200: 284).
            // Short launches: cut in two, their quads run half the chain and
            // then a merge, which costs more than the other half. Whole quads
            // where the longest sees at most 31 tiles; where the (quad, kv head)
            // pairs fill no more than a third of the compute units, at most 21,
            // and above that, up to 95, ranges of 8 tiles that the idle units
            // run beside each other. Graph replays over pools larger than the
            // caches, us at 8 tiles / the floor above / whole: 8-row verifies of
            // up to 450 keys at 15/5 heads x 64, 3 of them 9.9 / 10.2 / 10.2, 16
            // 11.9 / 14.5 / 12.8, 40 12.9 / 14.8 / 12.5; of up to 1000, 8 of them
            // 12.3 / 14.0 / 20; 16 prompts of up to 500 at 9/3 x 64 18.1 / 17.4 /
            // 15.2; 4 of up to 300 at 40/8 x 128 22.7 / 22.4 / 19.0.
            const bool few = quad_units <= kPlanCUs / 3;
            const double floor = longest < (few ? 22 : 32) ? longest : few && longest < 96 ? 8 : DP >= 128 ? 12 : 16;
            quad_w = std::max(floor, (double)visible / (2.0 * kPlanCUs));
            if (quad_w > 96) quad_w = std::max(96.0, (double)visible / (4.0 * kPlanCUs));
        }
    }
    // Partition counts per (sequence, quad), then at most two wide
    // workgroups per CU: rounding can leave a few more, and with every CU
    // holding two, those few land as a third on some CU, which then finishes
    // last. Partitions are merged, one at a time, in the quad whose ranges
    // grow the least. C2: 530 -> 510 workgroups, engine layer 42.1-42.3 us
    // against 42.7-42.9.
    std::vector<std::vector<int>> qparts(num_seqs);
    if (mixed || device) {
        int64_t total = 0;
        for (int s = 0; s < num_seqs; ++s) {
            const int nq = quads(s);
            qparts[s].resize(nq);
            for (int qd = 0; qd < nq; ++qd) {
                const int v = quad_visible(s, qd);
                const int n = std::max(1, (int)std::lround(v / quad_w));
                qparts[s][qd] = std::max<int>(n, ((int64_t)v + max_range - 1) / max_range);
                total += (int64_t)Hkv * qparts[s][qd];
            }
        }
        while (mixed && total > 2 * kPlanCUs) {
            int bs = -1, bq = -1;
            double best = 1e300;
            for (int s = 0; s < num_seqs; ++s)
                for (int qd = 0; qd < (int)qparts[s].size(); ++qd) {
                    const int n = qparts[s][qd], v = quad_visible(s, qd);
                    if (n <= 1 || (v + n - 2) / (n - 1) > max_range) continue;
                    const double grown = (double)v / (n - 1);
                    if (grown < best) {
                        best = grown;
                        bs = s;
                        bq = qd;
                    }
                }
            if (bs < 0) break;  // every quad is down to one range (or at the item limit)
            --qparts[bs][bq];
            total -= Hkv;
        }
    }
    auto quad_parts = [&](int s, int qd) { return qparts[s][qd]; };

    // First walk: sizes only.
    int64_t n_single = 0, n_coop = 0, n_wide = 0, n_loose = 0, n_merges = 0, n_slots = 0;
    for (int s = 0; s < num_seqs; ++s) {
        const int nct = col_tiles(s);
        if (!nct) continue;
        const bool narrow = nct == 1 || WT == 1;
        int Q;
        bool coop;
        const int nparts = partitions(s, narrow, Q, coop);
        const int width = narrow ? 1 : WT;
        const int ngroups = (nct + width - 1) / width;
        if (narrow) {
            if (coop) n_coop += (int64_t)U * nparts * Hkv * ngroups;
            else n_single += (int64_t)nparts * Hkv * ngroups;
        } else if (const int nq = quads(s)) {
            for (int qd = 0; qd < nq; ++qd) {
                const int n = quad_parts(s, qd);
                const int cols = std::min(nct, (qd + 1) * U * WT) - qd * U * WT;
                n_wide += (int64_t)Hkv * n * U;
                if (n > 1) {
                    n_slots += (int64_t)Hkv * n * cols;
                    n_merges += (int64_t)Hkv * cols;
                }
            }
            continue;
        } else if (ngroups >= U) {
            n_wide += (int64_t)nparts * Hkv * round_up(ngroups);
        } else {
            n_loose += (int64_t)nparts * Hkv * ngroups;
        }
        if (nparts > 1) {
            n_slots += (int64_t)Hkv * nparts * nct;
            n_merges += (int64_t)Hkv * nct;
        }
    }
    const int64_t n_narrow = round_up(n_single) + n_coop;
    n_wide += round_up(n_loose);
    const int64_t pstride = 16 * (int64_t)(mf::part_dstride_for(head_dim) + 2);
    counts[0] = n_narrow;
    counts[1] = n_wide;
    counts[2] = n_merges;
    counts[3] = n_slots * pstride;
    if (n_narrow + n_wide > items_capacity || n_merges > merges_capacity) return MF_ERR_WORKSPACE;
    if ((n_narrow + n_wide) > 0 && !items) return MF_ERR_ARG;
    if (n_merges > 0 && !merges) return MF_ERR_ARG;

    // Second walk: stage the items and write the merges. Column group gi of
    // a sequence owns partial slots from slot0 + gi*Hkv*nparts*width
    // (head-major, then partition, then its w tiles) and merge records from
    // merge0 + gi*Hkv*width.
    typedef std::array<int32_t, MF_PLAN_ITEM_INTS> Item;
    std::vector<Item> singles, coop_items, shared_items, loose_items;
    int64_t wm = 0, slots = 0;
    for (int s = 0; s < num_seqs; ++s) {
        const int nct = col_tiles(s);
        if (!nct) continue;
        const bool narrow = nct == 1 || WT == 1;
        const int tiles = (kv_lens[s] + 15) / 16;
        int Q;
        bool coop;
        const int nparts = partitions(s, narrow, Q, coop);
        const int width = narrow ? 1 : WT;
        const int ngroups = (nct + width - 1) / width;
        if (const int nq = narrow ? 0 : quads(s)) {
            // quad partitions: per (kv head, quad), each column group owns
            // n * w consecutive slots (partition-major) and w merge records;
            // a kv head's workgroups are consecutive (one XCD run)
            for (int h = 0; h < Hkv; ++h) {
                for (int qd = 0; qd < nq; ++qd) {
                    const int n = quad_parts(s, qd);
                    const int v = quad_visible(s, qd);
                    int64_t gslot[mf::kWaves], grec[mf::kWaves];
                    for (int k = 0; k < U; ++k) {
                        const int gi = qd * U + k;
                        gslot[k] = grec[k] = -1;
                        if (gi >= ngroups || n <= 1) continue;
                        const int w = std::min(WT, nct - gi * WT);
                        gslot[k] = slots;
                        slots += (int64_t)n * w;
                        grec[k] = wm;
                        for (int o2 = 0; o2 < w; ++o2, ++wm) {
                            int32_t* o = merges + wm * MF_PLAN_MERGE_INTS;
                            o[0] = s;
                            o[1] = h;
                            o[2] = gi * WT + o2;
                            o[3] = n;
                            o[4] = (int32_t)(gslot[k] + o2);
                            o[5] = w;
                            o[6] = cu_seqlens[s];
                            o[7] = cu_seqlens[s + 1] - cu_seqlens[s];
                        }
                    }
                    for (int p = 0; p < n; ++p) {
                        const int k0 = (int)((int64_t)p * v / n);
                        // v counts the keys of distinct positions that end the
                        // context; rows that share a position (the operator's
                        // non-causal queries) see more, so a device plan's last
                        // range runs to the context's end and the kernel stops
                        // where its rows do
                        const int k1 = device && p + 1 == n ? tiles : (int)((int64_t)(p + 1) * v / n);
                        for (int k = 0; k < U; ++k) {
                            const int gi = qd * U + k;
                            Item o{};
                            o[0] = s;
                            o[1] = h;
                            o[4] = k0;
                            o[5] = k1;
                            o[8] = cu_seqlens[s];
                            o[9] = cu_seqlens[s + 1] - cu_seqlens[s];
                            o[10] = kv_lens[s];
                            if (gi < ngroups) {
                                const int w = std::min(WT, nct - gi * WT);
                                o[2] = gi * WT;
                                o[3] = w;
                                o[6] = n > 1 ? (int32_t)(gslot[k] + (int64_t)p * w) : -1;
                                o[7] = n > 1 ? (int32_t)grec[k] : -1;
                            } else {  // padding: same keys, no columns, no partial slot
                                o[2] = (ngroups - 1) * WT;
                                o[6] = -1;
                                o[7] = -1;
                            }
                            shared_items.push_back(o);
                        }
                    }
                }
            }
            continue;
        }
        const int64_t slot0 = slots, merge0 = wm;
        const int32_t fp32_flag = narrow && unit_tiles > 0 && dtype != MF_F32 ? MF_PLAN_FP32_PARTIALS : 0;
        auto make = [&](int gi, int p, int h, int k0, int k1) {
            const int cg0 = gi * width;
            const int w = std::min(width, nct - cg0);
            Item o;
            o[0] = s;
            o[1] = h;
            o[2] = cg0;
            o[3] = w;
            o[4] = k0;
            o[5] = k1;
            o[6] = nparts > 1 ? (int32_t)(slot0 + (int64_t)gi * Hkv * nparts * width + ((int64_t)h * nparts + p) * w)
                              : -1;
            o[7] = nparts > 1 ? (int32_t)(merge0 + (int64_t)gi * Hkv * width + (int64_t)h * w) | fp32_flag : -1;
            o[8] = cu_seqlens[s];
            o[9] = cu_seqlens[s + 1] - cu_seqlens[s];
            o[10] = kv_lens[s];
            o[11] = 0;
            return o;
        };
        for (int p = 0; p < nparts; ++p) {
            const int k0 = part_begin(tiles, nparts, Q, coop, p);
            const int k1 = part_begin(tiles, nparts, Q, coop, p + 1);
            for (int hi = 0; hi < Hkv; ++hi) {
                // A device's decode units start one kv head on from the last
                // range's: with 8 heads workgroup b's head would otherwise be b
                // mod 8, its XCD's number, and an XCD that reads one head of
                // every row uses one channel in eight of its L2 (67 against 75
                // us, the 4 long sequences at 64-tile units).
                const int h = narrow && unit_tiles > 0 && !four ? (hi + p + s) % Hkv : hi;
                if (narrow) {
                    for (int gi = 0; gi < ngroups; ++gi) {
                        if (!coop) {
                            singles.push_back(make(gi, p, h, k0, k1));
                            continue;
                        }
                        // four waves on consecutive quarters of [k0, k1). In
                        // the unit holding a multi-row sequence's last tile (a
                        // verify pass: the boundary tile and the in-flight
                        // candidates, loaded key by key), the last wave counts
                        // MF_TAIL_WAVE_TILES more tiles than it has, so the
                        // others take them and the unit's waves reach its
                        // LDS combine together -- as far as a wave's
                        // block-table registers go.
                        const int n = k1 - k0;
                        const int rows = cu_seqlens[s + 1] - cu_seqlens[s];
                        const int extra = (k1 == tiles && rows > 1)
                                              ? std::min(MF_TAIL_WAVE_TILES, U * mf::kMaxItemTiles - n) : 0;
                        auto cut = [&](int w) {
                            return w >= U ? k1 : std::min(k1, k0 + (int)((int64_t)w * (n + extra) / U));
                        };
                        for (int w = 0; w < U; ++w) {
                            Item o = make(gi, p, h, cut(w), cut(w + 1));
                            o[11] = 1;
                            coop_items.push_back(o);
                        }
                    }
                } else if (ngroups >= U) {
                    for (int gi = 0; gi < round_up(ngroups); ++gi) {
                        Item o = make(std::min(gi, ngroups - 1), p, h, k0, k1);
                        if (gi >= ngroups) {  // padding: same keys, no columns, no partial slot
                            o[3] = 0;
                            o[6] = -1;
                            o[7] = -1;
                        }
                        shared_items.push_back(o);
                    }
                } else {
                    for (int gi = 0; gi < ngroups; ++gi) loose_items.push_back(make(gi, p, h, k0, k1));
                }
            }
        }
        if (nparts > 1) {
            for (int gi = 0; gi < ngroups; ++gi) {
                const int cg0 = gi * width;
                const int w = std::min(width, nct - cg0);
                const int64_t group_base = slot0 + (int64_t)gi * Hkv * nparts * width;
                for (int h = 0; h < Hkv; ++h) {
                    for (int o2 = 0; o2 < w; ++o2) {
                        int32_t* o = merges + wm * MF_PLAN_MERGE_INTS;
                        o[0] = s;
                        o[1] = h;
                        o[2] = cg0 + o2;
                        o[3] = nparts;
                        o[4] = (int32_t)(group_base + (int64_t)h * nparts * w + o2);
                        o[5] = w;
                        o[6] = cu_seqlens[s];
                        o[7] = (cu_seqlens[s + 1] - cu_seqlens[s]) | fp32_flag;
                        ++wm;
                    }
                }
            }
            slots += (int64_t)Hkv * nparts * nct;
        }
    }
    // Longest first: the hardware hands out workgroups in order as slots free
    // up, so the last round of the grid is made of the short remainder
    // partitions instead of a few long ones. Items that run alone are sorted
    // and then cut into workgroups (the last padded with empty items); all
    // workgroups are ordered by their longest item. Stable, so equal lengths
    // keep their heads-adjacent order.
    auto len = [](const Item& o) { return o[5] - o[4]; };
    auto longer = [&](const Item& x, const Item& y) { return len(x) > len(y); };
    auto pad_to_workgroups = [&](std::vector<Item>& v) {
        std::stable_sort(v.begin(), v.end(), longer);
        while (v.size() % U) {
            Item o{};
            o[6] = -1;
            o[7] = -1;
            v.push_back(o);
        }
    };
    auto unit_len = [&](const Item* u) {
        int l = 0;
        for (int w = 0; w < U; ++w) l = std::max(l, len(u[w]));
        return l;
    };
    auto emit = [&](std::vector<const Item*>& units, int64_t wi) {
        std::stable_sort(units.begin(), units.end(),
                         [&](const Item* x, const Item* y) { return unit_len(x) > unit_len(y); });
        for (const Item* u : units)
            for (int w = 0; w < U; ++w, ++wi) std::copy(u[w].begin(), u[w].end(), items + wi * MF_PLAN_ITEM_INTS);
    };
    pad_to_workgroups(singles);
    pad_to_workgroups(loose_items);
    std::vector<const Item*> nunits, wunits;
    for (size_t i = 0; i < coop_items.size(); i += U) nunits.push_back(&coop_items[i]);
    for (size_t i = 0; i < singles.size(); i += U) nunits.push_back(&singles[i]);
    for (size_t i = 0; i < shared_items.size(); i += U) wunits.push_back(&shared_items[i]);
    for (size_t i = 0; i < loose_items.size(); i += U) wunits.push_back(&loose_items[i]);
    emit(nunits, 0);
    // A wide item's work: its tiles up to the last one its last column sees
    // (causal), a workgroup's the most of its four.
    auto item_work = [&](const Item& o) -> int64_t {
        const int ncols = o[9] * G;
        const int last_col = std::min((o[2] + o[3]) * 16, ncols) - 1;
        if (o[3] <= 0 || last_col < 0) return 0;
        const int last_pos = o[10] - o[9] + last_col / G;
        return std::max(0, std::min(o[5], last_pos / 16 + 1) - o[4]);
    };
    auto unit_work = [&](const Item* u) {
        int64_t l = 0;
        for (int w = 0; w < U; ++w) l = std::max(l, item_work(u[w]));
        return l;
    };
    if (MF_WIDE_XCD) {
        // Runs of workgroups on one key range, most work first, are dealt
        // to the queue with the least work so far; each queue then runs its
        // workgroups most work first, and the queues are interleaved.
        constexpr int X = 8;
        const size_t nu = wunits.size();
        std::vector<int64_t> work(nu);
        for (size_t i = 0; i < nu; ++i) work[i] = unit_work(wunits[i]);
        auto same_range = [&](size_t x, size_t y) {
            const Item& a = wunits[x][0];
            const Item& b = wunits[y][0];
            // one key range; in a mixed plan one (sequence, kv head), whose
            // quads' ranges overlap
            return a[0] == b[0] && a[1] == b[1] && (mixed || device || (a[4] == b[4] && a[5] == b[5]));
        };
        // run r holds units [run_begin[r], run_begin[r + 1])
        std::vector<size_t> run_begin;
        std::vector<int64_t> run_work;
        for (size_t i = 0; i < nu; ++i) {
            if (i >= shared_items.size() / U || run_begin.empty() || !same_range(i - 1, i)) {
                run_begin.push_back(i);
                run_work.push_back(0);
            }
            run_work.back() += work[i];
        }
        const size_t nruns = run_begin.size();
        run_begin.push_back(nu);
        std::vector<size_t> order(nruns);
        for (size_t i = 0; i < nruns; ++i) order[i] = i;
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return run_work[x] > run_work[y]; });
        // queue x holds exactly the workgroups at wide positions x mod 8; a
        // run that no queue has room for is split over the roomiest ones
        std::vector<size_t> queue[X];
        int64_t load[X] = {};
        for (auto& q : queue) q.reserve(nu / X + 1);
        auto room = [&](int x) { return (int64_t)(nu / X + (x < (int)(nu % X) ? 1 : 0)) - (int64_t)queue[x].size(); };
        for (size_t ri : order) {
            size_t i = run_begin[ri];
            const size_t end = run_begin[ri + 1];
            while (i < end) {
                int best = -1;
                for (int x = 0; x < X; ++x)
                    if (room(x) >= (int64_t)(end - i) && (best < 0 || load[x] < load[best])) best = x;
                if (best < 0) {
                    for (int x = 0; x < X; ++x)
                        if (best < 0 || room(x) > room(best)) best = x;
                }
                const size_t take = std::min<size_t>(end - i, (size_t)room(best));
                for (size_t t = 0; t < take; ++t, ++i) {
                    queue[best].push_back(i);
                    load[best] += work[i];
                }
            }
        }
        for (auto& q : queue)
            std::stable_sort(q.begin(), q.end(), [&](size_t x, size_t y) { return work[x] > work[y]; });
        int64_t wi = n_narrow;
        for (size_t k = 0;; ++k) {
            bool any = false;
            for (int x = 0; x < X; ++x) {
                if (k >= queue[x].size()) continue;
                any = true;
                const Item* u = wunits[queue[x][k]];
                for (int w = 0; w < U; ++w, ++wi) std::copy(u[w].begin(), u[w].end(), items + wi * MF_PLAN_ITEM_INTS);
            }
            if (!any) break;
        }
    } else {
        emit(wunits, n_narrow);
    }
    return MF_OK;
}
}  // namespace

extern "C" int mf_attention_plan(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                 int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                 int partition_tiles, int32_t* items, int64_t items_capacity,
                                 int32_t* merges, int64_t merges_capacity, int64_t* counts) {
    return attention_plan(num_seqs, cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype,
                          partition_tiles, 0, true, items, items_capacity, merges, merges_capacity, counts);
}

extern "C" int mf_attention_plan_device(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                        int num_q_heads, int num_kv_heads, int head_dim, int dtype, int num_cus,
                                        int32_t* items, int64_t items_capacity, int32_t* merges,
                                        int64_t merges_capacity, int64_t* counts) {
    if (num_cus <= 0) return MF_ERR_ARG;
    return attention_plan(num_seqs, cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype, 0, num_cus, true,
                          items, items_capacity, merges, merges_capacity, counts);
}

extern "C" int mf_attention_plan_merge_free(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                            int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                            int num_cus, int32_t* items, int64_t items_capacity, int32_t* merges,
                                            int64_t merges_capacity, int64_t* counts) {
    if (num_cus <= 0) return MF_ERR_ARG;
    return attention_plan(num_seqs, cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype, 0, num_cus, false,
                          items, items_capacity, merges, merges_capacity, counts);
}

extern "C" int mf_attention_plan4(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens, int num_q_heads,
                                  int num_kv_heads, int head_dim, int dtype, int num_cus, int32_t* items,
                                  int64_t items_capacity, int32_t* merges, int64_t merges_capacity, int64_t* counts) {
    if (num_cus <= 0) return MF_ERR_ARG;
    try {
        return attention_plan(num_seqs, cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype, 0, num_cus,
                              true, items, items_capacity, merges, merges_capacity, counts, /*four=*/true);
    } catch (const std::exception&) {  // no memory for a plan of this size
        return MF_ERR_ARG;
    }
}

// Slice plan for a large decode launch (attn_slice_kernel). The sequences'
// 16-key tiles, in sequence order, are cut into slices of about
// total / (num_cus * MF_SLICE_WAVES_PER_CU / Hkv) tiles, so one wave per
// (slice, kv head) fills the GPU exactly once at one workgroup per CU. A slice holds at most MF_SLICE_MAX_SEGMENTS
// segments and MF_SLICE_MAX_TILES tiles once each segment is padded to a
// multiple of the kernel's ring depth; a workload whose even share would
// exceed that gets more slices (a second round). A sequence cut across
// slices leaves one partial per piece and kv head, merged afterwards.
extern "C" int mf_attention_plan_slices(int num_seqs, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                        int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                        int num_cus, int min_tiles_per_wave, int32_t* slices,
                                        int64_t slices_capacity, int32_t* merges, int64_t merges_capacity,
                                        int64_t* counts) {
    if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || !counts || num_cus <= 0 ||
        min_tiles_per_wave < 0)
        return MF_ERR_ARG;
    const int64_t resident_waves = (int64_t)num_cus * MF_SLICE_WAVES_PER_CU;
    if (num_q_heads % num_kv_heads) return MF_ERR_ARG;
    if (num_seqs > 0 && (!cu_seqlens || !kv_lens)) return MF_ERR_ARG;
    const int DP = mf::padded_head_dim(dtype, head_dim);
    if (!mf::dtype_ok(dtype) || !DP) return MF_ERR_UNSUPPORTED;
    const int G = num_q_heads / num_kv_heads;
    const int Hkv = num_kv_heads;
    counts[0] = counts[1] = counts[2] = counts[3] = 0;
    // Decode only: one query row per sequence, whose heads fit one column
    // tile, and head_dim at one of the kernel's sizes.
    if (DP != head_dim || G > 16) return MF_ERR_UNSUPPORTED;
    int64_t total = 0;
    for (int s = 0; s < num_seqs; ++s) {
        const int qlen = cu_seqlens[s + 1] - cu_seqlens[s];
        if (qlen < 0) return MF_ERR_ARG;
        if (kv_lens[s] <= 0 || qlen == 0) continue;
        if (qlen != 1) return MF_ERR_UNSUPPORTED;
        total += (kv_lens[s] + 15) / 16;
    }
    // Launches whose tiles give each resident wave fewer than
    // min_tiles_per_wave get no slice plan (counts stay zero): at
    // MF_SLICE_MIN_TILES and below, per-range items fit them in one round.
    if (total == 0 || total * Hkv < (int64_t)min_tiles_per_wave * resident_waves) return MF_OK;

    // Slices per round fill the GPU once; a workload whose even share would
    // not fit one slice runs whole rounds of equal slices (a round with only
    // a few slices would leave the GPU idle for its whole length). A slice's
    // real tiles stay below MF_SLICE_MAX_TILES by enough for the padding of
    // sixteen segments, so padding rarely closes a slice early.
    constexpr int NB = MF_NARROW_DEPTH;
    const int64_t base_slices = std::max<int64_t>(1, resident_waves / Hkv);
    const int64_t fill_cap = mf::kSliceMaxTiles - 16 * (NB - 1);
    const int64_t rounds = (total + base_slices * fill_cap - 1) / (base_slices * fill_cap);
    const int64_t want = rounds * base_slices;
    // slice i carries total / want tiles, one more for the first total % want
    const int64_t share = total / want, extra = total % want;

    // First walk: cut the slices (segment = sequence, kt0, kt1).
    struct Seg { int s, kt0, kt1; };
    std::vector<Seg> segs;
    std::vector<int64_t> begins;  // first segment of each slice
    std::vector<int> padded;      // padded tiles of each slice
    int64_t cur_real = 0, target = 0;
    int cur_pad = 0, cur_n = 0;
    auto open_slice = [&]() {
        target = std::max<int64_t>(1, share + ((int64_t)begins.size() < extra ? 1 : 0));
        begins.push_back((int64_t)segs.size());
        padded.push_back(0);
        cur_real = 0;
        cur_pad = 0;
        cur_n = 0;
    };
    open_slice();
    for (int s = 0; s < num_seqs; ++s) {
        const int qlen = cu_seqlens[s + 1] - cu_seqlens[s];
        if (kv_lens[s] <= 0 || qlen == 0) continue;
        const int T = (kv_lens[s] + 15) / 16;
        int kt = 0;
        while (kt < T) {
            const int64_t room_pad = mf::kSliceMaxTiles - cur_pad;
            if (cur_n == mf::kSliceMaxSegments || cur_real >= target || room_pad < NB) {
                open_slice();
                continue;
            }
            const int64_t take = std::min<int64_t>({(int64_t)(T - kt), target - cur_real, room_pad / NB * NB});
            segs.push_back({s, kt, (int)(kt + take)});
            cur_real += take;
            cur_pad += (int)((take + NB - 1) / NB * NB);
            padded.back() = cur_pad;
            ++cur_n;
            kt += (int)take;
        }
    }
    if (padded.back() == 0) {  // a slice opened after the last segment
        begins.pop_back();
        padded.pop_back();
    }
    const int64_t n_slices = (int64_t)begins.size();
    const int64_t n_segs = (int64_t)segs.size();

    // Pieces per sequence: slot ranges and merge records for split ones.
    std::vector<int> pieces(num_seqs, 0);
    for (const Seg& g : segs) ++pieces[g.s];
    int64_t n_merges = 0, n_slots = 0;
    for (int s = 0; s < num_seqs; ++s)
        if (pieces[s] > 1) {
            n_merges += Hkv;
            n_slots += (int64_t)Hkv * pieces[s];
        }
    counts[0] = n_slices;
    counts[1] = n_segs;
    counts[2] = n_merges;
    counts[3] = n_slots * 16 * (int64_t)(mf::part_dstride_for(head_dim) + 2);
    if (n_slices + n_segs > slices_capacity || n_merges > merges_capacity) return MF_ERR_WORKSPACE;
    if (!slices || (n_merges > 0 && !merges)) return MF_ERR_ARG;

    constexpr int R = MF_SLICE_INTS;
    for (int64_t i = 0; i < n_slices; ++i) {
        int32_t* o = slices + i * R;
        const int64_t end = i + 1 < n_slices ? begins[i + 1] : n_segs;
        std::fill(o, o + R, 0);
        o[0] = (int32_t)begins[i];
        o[1] = (int32_t)(end - begins[i]);
        o[2] = padded[i];
    }
    std::vector<int64_t> slot0(num_seqs, -1);
    int64_t slots = 0, wm = 0;
    for (int s = 0; s < num_seqs; ++s) {
        if (pieces[s] <= 1) continue;
        slot0[s] = slots;
        for (int h = 0; h < Hkv; ++h) {
            int32_t* o = merges + (wm++) * MF_PLAN_MERGE_INTS;
            o[0] = s;
            o[1] = h;
            o[2] = 0;
            o[3] = pieces[s];
            o[4] = (int32_t)(slots + (int64_t)h * pieces[s]);
            o[5] = 1;
            o[6] = cu_seqlens[s];
            o[7] = 1;
        }
        slots += (int64_t)Hkv * pieces[s];
    }
    std::vector<int> part(num_seqs, 0);
    for (int64_t i = 0; i < n_segs; ++i) {
        const Seg& g = segs[i];
        int32_t* o = slices + (n_slices + i) * R;
        o[0] = g.s;
        o[1] = g.kt0;
        o[2] = g.kt1;
        o[3] = cu_seqlens[g.s];
        o[4] = kv_lens[g.s];
        o[5] = (int32_t)slot0[g.s];
        o[6] = pieces[g.s];
        o[7] = part[g.s]++;
    }
    return MF_OK;
}

namespace {
int paged_attention_impl(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, const void* k_pool, const void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens,
    const int32_t* kv_lens, const int64_t* positions, const int32_t* row_map,
    const int32_t* pool_lens, const void* new_k, const void* new_v, int64_t new_stride_row,
    int64_t new_stride_head, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide,
    const int32_t* plan_merges, int64_t num_merges, float* partials, int64_t partials_floats,
    int32_t* merge_counters, const int32_t* device_counts, mf_stream_t stream, bool sliced = false,
    const int64_t* write_slots = nullptr, int64_t write_rows = 0, int64_t write_num_slots = 0,
    bool tail_inflight = false, const mf_scoring* scoring = nullptr) {
    using namespace mf;
    if (!(std::fabs(scale) < INFINITY)) return MF_ERR_ARG;  // NaN or infinite
    if (!dtype_ok(dtype) || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        block_size <= 0 || num_items_narrow < 0 || num_items_wide < 0 || num_merges < 0)
        return MF_ERR_ARG;
    const int DP = padded_head_dim(dtype, head_dim);
    if (!DP) return MF_ERR_UNSUPPORTED;
    // A call may carry only items (partials left for a later merge-only call)
    // or only merges; both are how a caller times the two kernels apart.
    if (num_items_narrow + num_items_wide == 0 && num_merges == 0 && write_rows == 0) return MF_OK;
    if (!q || !out || !k_pool || !v_pool || !block_tables || !cu_seqlens || !kv_lens || !positions)
        return MF_ERR_ARG;
    if (num_items_narrow + num_items_wide > 0 && !plan_items) return MF_ERR_ARG;
    // Range-plan items run in workgroups of four and a wave loads its item
    // before its count check: both counts are whole workgroups, as plans make
    // them (a slice plan's counts are slices and segments).
    if (!sliced && ((num_items_narrow % kWaves) || (num_items_wide % kWaves))) return MF_ERR_ARG;
    if (pool_lens && (!new_k || !new_v)) return MF_ERR_ARG;
    if (num_merges > 0 && (!plan_merges || !partials || partials_floats <= 0)) return MF_ERR_WORKSPACE;
    // 16-byte row loads need 16-byte aligned rows.
    const int es = dtype_size(dtype);
    const int64_t epl = 16 / es;
    const int64_t strides[] = {q_stride_row, q_stride_head, pool_stride_block, pool_stride_slot,
                               pool_stride_head};
    for (int64_t st : strides)
        if (st % epl) return MF_ERR_ARG;
    if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) return MF_ERR_ARG;
    if (pool_lens && ((new_stride_row % epl) || (new_stride_head % epl) ||
                      (((uintptr_t)new_k | (uintptr_t)new_v) & 15)))
        return MF_ERR_ARG;
    const int out_align = std::min(16, 4 * (DP / 16) * es);
    if ((out_stride_row * es) % out_align || (out_stride_head * es) % out_align ||
        ((uintptr_t)out % out_align))
        return MF_ERR_ARG;

    ScoredArgs a{};
    a.q = (const char*)q;
    a.q_sr = q_stride_row;
    a.q_sh = q_stride_head;
    a.out = (char*)out;
    a.o_sr = out_stride_row;
    a.o_sh = out_stride_head;
    a.k_pool = (const char*)k_pool;
    a.v_pool = (const char*)v_pool;
    a.p_sb = pool_stride_block;
    a.p_ss = pool_stride_slot;
    a.p_sh = pool_stride_head;
    a.block_size = block_size;
    a.block_tables = block_tables;
    a.bt_stride = block_table_stride;
    a.cu_seqlens = cu_seqlens;
    a.kv_lens = kv_lens;
    a.positions = positions;
    a.row_map = row_map;
    a.pool_lens = pool_lens;
    a.new_k = (const char*)new_k;
    a.new_v = (const char*)new_v;
    a.n_sr = new_stride_row;
    a.n_sh = new_stride_head;
    a.G = num_q_heads / num_kv_heads;
    a.head_dim = head_dim;
    // Scores are scaled inside the exponent, which needs a positive factor:
    // a negative scale flips the sign of Q instead (exact), and a zero scale
    // becomes 2^-100, for which every 2^(s * scale - m) rounds to exactly 1,
    // the uniform weights a zero scale gives.
    a.q_sign = scale < 0.f ? (es == 4 ? 0x80000000u : 0x80008000u) : 0u;
    a.scale_log2 = scale == 0.f ? 0x1p-100f : std::fabs(scale) * 1.4426950408889634f;
    a.inv_scale_log2 = 1.f / a.scale_log2;
    a.partials = partials;
    a.part_dstride = part_dstride_for(head_dim);
    a.merges = plan_merges;
    a.counters = num_merges > 0 ? merge_counters : nullptr;
    a.num_kv_heads = num_kv_heads;
    const bool fast = block_size == 16 && head_dim == DP;
    hipStream_t st = (hipStream_t)stream;
    if (tail_inflight) {
        if (!new_k || !new_v || row_map || pool_lens || write_rows < 0 || write_num_slots < 0) return MF_ERR_ARG;
        if (write_rows > 0 && !write_slots) return MF_ERR_ARG;
        if ((new_stride_row % epl) || (new_stride_head % epl) || (((uintptr_t)new_k | (uintptr_t)new_v) & 15))
            return MF_ERR_ARG;
        if (!fast) {
            // other block sizes and padded head_dims: the write, then the
            // attention reading every key from the pool (same result, two launches)
            if (write_rows > 0) {
                if (int sw = mf_kv_write(new_k, new_v, dtype, new_stride_row, new_stride_head, write_slots,
                                         write_rows, const_cast<void*>(k_pool), const_cast<void*>(v_pool), dtype,
                                         pool_stride_block, pool_stride_slot, pool_stride_head, block_size,
                                         write_num_slots, num_kv_heads, head_dim, stream))
                    return sw;
            }
            tail_inflight = false;
        } else {
            // the copy: 16-byte pieces of every new row's K and V, about four
            // per thread of the copy workgroups
            const int64_t pieces = write_rows * 2 * num_kv_heads * (head_dim * es / 16);
            if (pieces > INT_MAX / 2) return MF_ERR_ARG;
            a.w_slots = write_slots;
            a.w_rows = (int)write_rows;
            a.w_num_slots = write_num_slots;
            a.w_blocks = pieces > 0 ? (int)std::min<int64_t>(1024, (pieces + 1023) / 1024) : 0;
        }
    }

    if (sliced && (!fast || row_map || pool_lens || merge_counters || device_counts || tail_inflight))
        return MF_ERR_UNSUPPORTED;
    if (scoring) {
        if (sliced || merge_counters) return MF_ERR_UNSUPPORTED;
        if (int se = set_scoring(a, *scoring)) return se;
        return launch_scored(dtype, DP, tail_inflight, a, plan_items, num_items_narrow, num_items_wide, plan_merges,
                             num_merges, fast, device_counts, st);
    }
#define MF_ATTN_CASE(DT, DPV)                                                                  \
    if (dtype == DT && DP == DPV)                                                              \
        return sliced ? launch_slices<DT, DPV>(a, plan_items, num_items_narrow, num_kv_heads,  \
                                               plan_merges, num_merges, st)                    \
                      : (tail_inflight ? launch_attention<DT, DPV, true>(a, plan_items, num_items_narrow, \
                                                                         num_items_wide, plan_merges, num_merges, \
                                                                         fast, device_counts, st) \
                                       : launch_attention<DT, DPV>(a, plan_items, num_items_narrow, num_items_wide, \
                                                                   plan_merges, num_merges, fast, device_counts, st));
    MF_ATTN_CASE(MF_F32, 16)
    MF_ATTN_CASE(MF_F32, 32)
    MF_ATTN_CASE(MF_F32, 64)
    MF_ATTN_CASE(MF_F32, 128)
    MF_ATTN_CASE(MF_BF16, 32)
    MF_ATTN_CASE(MF_BF16, 64)
    MF_ATTN_CASE(MF_BF16, 128)
    MF_ATTN_CASE(MF_BF16, 256)
    MF_ATTN_CASE(MF_F16, 32)
    MF_ATTN_CASE(MF_F16, 64)
    MF_ATTN_CASE(MF_F16, 128)
    MF_ATTN_CASE(MF_F16, 256)
#undef MF_ATTN_CASE
    return MF_ERR_UNSUPPORTED;
}
}  // namespace

extern "C" int mf_paged_attention(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, const void* k_pool, const void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens,
    const int32_t* kv_lens, const int64_t* positions, const int32_t* row_map,
    const int32_t* pool_lens, const void* new_k, const void* new_v, int64_t new_stride_row,
    int64_t new_stride_head, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide,
    const int32_t* plan_merges, int64_t num_merges, float* partials, int64_t partials_floats,
    int32_t* merge_counters, mf_stream_t stream) {
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                row_map, pool_lens, new_k, new_v, new_stride_row, new_stride_head, num_q_heads,
                                num_kv_heads, head_dim, scale, plan_items, num_items_narrow, num_items_wide,
                                plan_merges, num_merges, partials, partials_floats, merge_counters, nullptr,
                                stream);
}

extern "C" int mf_paged_attention_slices(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, const void* k_pool, const void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens,
    const int32_t* kv_lens, const int64_t* positions, int num_q_heads, int num_kv_heads, int head_dim,
    float scale, const int32_t* slices, int64_t num_slices, int64_t num_segments,
    const int32_t* plan_merges, int64_t num_merges, float* partials, int64_t partials_floats,
    mf_stream_t stream) {
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                nullptr, nullptr, nullptr, nullptr, 0, 0, num_q_heads, num_kv_heads, head_dim,
                                scale, slices, num_slices, num_segments, plan_merges, num_merges, partials,
                                partials_floats, nullptr, nullptr, stream, /*sliced=*/true);
}

extern "C" int mf_paged_attention_counted(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, const void* k_pool, const void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens,
    const int32_t* kv_lens, const int64_t* positions, const int32_t* row_map,
    const int32_t* pool_lens, const void* new_k, const void* new_v, int64_t new_stride_row,
    int64_t new_stride_head, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    const int32_t* plan_items, int64_t capacity_narrow, int64_t capacity_wide,
    const int32_t* plan_merges, int64_t capacity_merges, const int32_t* device_counts, float* partials,
    int64_t partials_floats, mf_stream_t stream) {
    if (!device_counts) return MF_ERR_ARG;
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                row_map, pool_lens, new_k, new_v, new_stride_row, new_stride_head, num_q_heads,
                                num_kv_heads, head_dim, scale, plan_items, capacity_narrow, capacity_wide,
                                plan_merges, capacity_merges, partials, partials_floats, nullptr,
                                device_counts, stream);
}

extern "C" int mf_paged_attention_kv_write(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, void* k_pool, void* v_pool, int64_t pool_stride_block,
    int64_t pool_stride_slot, int64_t pool_stride_head, int block_size, const int32_t* block_tables,
    int64_t block_table_stride, const int32_t* cu_seqlens, const int32_t* kv_lens, const int64_t* positions,
    const void* new_k, const void* new_v, int64_t new_stride_row, int64_t new_stride_head,
    const int64_t* slot_mapping, int64_t num_new_rows, int64_t num_slots, int num_q_heads, int num_kv_heads,
    int head_dim, float scale, const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide,
    const int32_t* plan_merges, int64_t num_merges, const int32_t* device_counts, float* partials,
    int64_t partials_floats, mf_stream_t stream) {
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                nullptr, nullptr, new_k, new_v, new_stride_row, new_stride_head, num_q_heads,
                                num_kv_heads, head_dim, scale, plan_items, num_items_narrow, num_items_wide,
                                plan_merges, num_merges, partials, partials_floats, nullptr, device_counts,
                                stream, /*sliced=*/false, slot_mapping, num_new_rows, num_slots,
                                /*tail_inflight=*/true);
}

extern "C" int mf_paged_attention_scored(
    const mf_scoring* scoring, const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out,
    int64_t out_stride_row, int64_t out_stride_head, int dtype, void* k_pool, void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens, const int32_t* kv_lens,
    const int64_t* positions, const int32_t* row_map, const int32_t* pool_lens, const void* new_k,
    const void* new_v, int64_t new_stride_row, int64_t new_stride_head, const int64_t* slot_mapping,
    int64_t num_new_rows, int64_t num_slots, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide, const int32_t* plan_merges,
    int64_t num_merges, const int32_t* device_counts, float* partials, int64_t partials_floats,
    mf_stream_t stream) {
    if (!scoring) return MF_ERR_ARG;
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                row_map, pool_lens, new_k, new_v, new_stride_row, new_stride_head, num_q_heads,
                                num_kv_heads, head_dim, scale, plan_items, num_items_narrow, num_items_wide,
                                plan_merges, num_merges, partials, partials_floats, nullptr, device_counts,
                                stream, /*sliced=*/false, slot_mapping, slot_mapping ? num_new_rows : 0,
                                slot_mapping ? num_slots : 0, /*tail_inflight=*/slot_mapping != nullptr, scoring);
}

// ------------------------------------------------------- no-allocation entry
//
// mf_paged_attention for callers that cannot allocate device memory: the
// split-K partials go to `scratch`, a library-owned device array that every
// GPU holding this code object keeps until the process ends. In host code the
// array's name is only a stand-in for the symbol; its device address, which
// differs per GPU, comes from hipGetSymbolAddress on the first call on each
// device and is the only form host code ever passes to a kernel. Nothing in
// it needs clearing between calls (every partial slot is written before the
// merge reads it), and calls that overlap on one GPU race on it.
static __device__ __align__(256) float scratch[MF_NOALLOC_PARTIALS_FLOATS];

namespace {
constexpr int kMaxScratchDevices = 64;
std::atomic<float*> g_scratch_ptr[kMaxScratchDevices];
std::mutex g_scratch_mu;

// Device address of the current device's `scratch`, looked up once per device.
int scratch_for_current_device(float** out) {
    int dev = -1;
    hipError_t err = hipGetDevice(&dev);
    if (err != hipSuccess) {
        mf::set_last_hip_error((int)err);
        return MF_ERR_HIP;
    }
    if (dev < 0 || dev >= kMaxScratchDevices) return MF_ERR_UNSUPPORTED;
    float* p = g_scratch_ptr[dev].load(std::memory_order_acquire);
    if (!p) {
        std::lock_guard<std::mutex> lock(g_scratch_mu);
        p = g_scratch_ptr[dev].load(std::memory_order_relaxed);
        if (!p) {
            void* addr = nullptr;
            err = hipGetSymbolAddress(&addr, HIP_SYMBOL(scratch));
            if (err != hipSuccess || !addr) {
                mf::set_last_hip_error((int)err);
                return MF_ERR_HIP;
            }
            p = (float*)addr;
            g_scratch_ptr[dev].store(p, std::memory_order_release);
        }
    }
    *out = p;
    return MF_OK;
}
}  // namespace

extern "C" int mf_paged_attention_noalloc(
    const void* q, int64_t q_stride_row, int64_t q_stride_head, void* out, int64_t out_stride_row,
    int64_t out_stride_head, int dtype, const void* k_pool, const void* v_pool,
    int64_t pool_stride_block, int64_t pool_stride_slot, int64_t pool_stride_head, int block_size,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* cu_seqlens,
    const int32_t* kv_lens, const int64_t* positions, const int32_t* row_map,
    const int32_t* pool_lens, const void* new_k, const void* new_v, int64_t new_stride_row,
    int64_t new_stride_head, int num_q_heads, int num_kv_heads, int head_dim, float scale,
    const int32_t* plan_items, int64_t num_items_narrow, int64_t num_items_wide,
    const int32_t* plan_merges, int64_t num_merges, int64_t partials_floats, mf_stream_t stream) {
    // sizes first: a plan that needs more than the array is refused before
    // anything touches the device
    if (partials_floats < 0) return MF_ERR_ARG;
    if (partials_floats > MF_NOALLOC_PARTIALS_FLOATS) return MF_ERR_WORKSPACE;
    float* partials = nullptr;
    if (int st = scratch_for_current_device(&partials)) return st;
    return paged_attention_impl(q, q_stride_row, q_stride_head, out, out_stride_row, out_stride_head, dtype,
                                k_pool, v_pool, pool_stride_block, pool_stride_slot, pool_stride_head,
                                block_size, block_tables, block_table_stride, cu_seqlens, kv_lens, positions,
                                row_map, pool_lens, new_k, new_v, new_stride_row, new_stride_head, num_q_heads,
                                num_kv_heads, head_dim, scale, plan_items, num_items_narrow, num_items_wide,
                                plan_merges, num_merges, partials, MF_NOALLOC_PARTIALS_FLOATS, nullptr,
                                nullptr, stream);
}
