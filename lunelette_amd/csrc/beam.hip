// Beam search: the next hypotheses over beams and vocabulary (lh_beam_select) and the
// paged caches' reordering after it (lh_beam_reorder).
//
// A candidate's score is s + (x - m) - ln Z with m and Z of its beam's row. Its order
// inside a row is that of its logit, so a row's best `keep` tokens by logit are all
// that can be among the group's best. One pass over the logits, as for log
// probabilities, gives every part of a row its range and its best tokens; a second
// launch of a workgroup a group forms the scores in 64 bits and orders the few of them
// that can be among the best.
#include "lh_paged.h"
#include "lh_serving.h"
#include "lh_topk.h"

namespace lh {

// A candidate as one 128-bit number whose larger value is the better place: the score,
// then the lower beam (6 bits), the larger logit (its rank, 32), the lower id (24). 0
// is no candidate: no score above -Inf has a rank of 0.
struct Place {
    uint64_t score, rest;
};

__device__ __forceinline__ bool operator>(const Place& a, const Place& b)
{
    return a.score != b.score ? a.score > b.score : a.rest > b.rest;
}

__device__ __forceinline__ uint64_t score_rank(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}

__device__ __forceinline__ double rank_score(uint64_t rank)
{
    return __builtin_bit_cast(double, rank >> 63 ? rank & ~((uint64_t)1 << 63) : ~rank);
}

__device__ __forceinline__ Place place_of(double score, uint32_t beam, uint32_t logit,
    uint32_t id)
{
    return {score_rank(score), (uint64_t)(63 - beam) << 56 | (uint64_t)logit << 24 |
        (0xffffffu - id)};
}

template <int J>
__device__ __forceinline__ Place exchange(Place p, uint32_t lane, bool larger)
{
    const Place other = {
        (uint64_t)xor_word<J>((uint32_t)(p.score >> 32), lane) << 32 |
            xor_word<J>((uint32_t)p.score, lane),
        (uint64_t)xor_word<J>((uint32_t)(p.rest >> 32), lane) << 32 |
            xor_word<J>((uint32_t)p.rest, lane)};
    return (other > p) == larger ? other : p;
}

template <int J>
__device__ __forceinline__ Place half_merge(Place p, uint32_t lane, bool falling)
{
    p = exchange<J>(p, lane, ((lane & J) == 0) == falling);
    if constexpr (J > 1) {
        p = half_merge<J / 2>(p, lane, falling);
    }
    return p;
}

// The 64 lanes' places in order, as sort_keys.
__device__ __forceinline__ Place sort_places(Place p, uint32_t lane, bool falling)
{
    p = half_merge<1>(p, lane, (lane & 2) != 0);
    p = half_merge<2>(p, lane, (lane & 4) != 0);
    p = half_merge<4>(p, lane, (lane & 8) != 0);
    p = half_merge<8>(p, lane, (lane & 16) != 0);
    p = half_merge<16>(p, lane, (lane & 32) != 0);
    return half_merge<32>(p, lane, falling);
}

__device__ __forceinline__ Place merge_places(Place best, Place rising, uint32_t lane)
{
    return half_merge<32>(best > rising ? best : rising, lane, true);
}

// PLACES: candidates that reach the group's bound at most, `keep` of as many lists. FEW:
// candidates that are counted, not sorted.
enum { PLACES = LH_BEAMS * LH_BEAMS, FEW = 128, SHARE = FEW * FEW / (64 * WAVES) };

struct BeamArgs {
    lh_beam_choice c;
    Range* ranges;      // [row][part]
    uint64_t* keys;     // [row][part][keep]
    uint32_t parts;
};

// A beam whose logits count: not finished and with a score above -Inf (a NaN too, which
// the join refuses).
__device__ __forceinline__ bool scans(const lh_beam_choice& c, size_t row)
{
    return !(c.done && c.done[row]) && !(c.scores[row] == -__builtin_inff());
}

// grid (parts, rows).
__global__ void __launch_bounds__(64 * WAVES)
k_beam_parts(BeamArgs a)
{
    __shared__ PartShared sh;
    const lh_beam_choice& c = a.c;
    const size_t row = blockIdx.y;
    if (!scans(c, row)) {
        return;
    }
    Range r;
    uint64_t key;
    scan_part<false>(sh, c.logits + row * c.stride, c.vocab, c.keep, blockIdx.x, a.parts, r, key);
    if (threadIdx.x >= 64) {
        return;
    }
    const size_t at = row * a.parts + blockIdx.x;
    if (threadIdx.x == 0) {
        a.ranges[at] = r;
    }
    if (threadIdx.x < c.keep) {
        a.keys[at * c.keep + threadIdx.x] = key;
    }
}

struct BeamShared {
    double base[LH_BEAMS], log_z[LH_BEAMS];
    float most[LH_BEAMS];
    uint32_t kind[LH_BEAMS], bad, count, rank[FEW];
    Place bound, lists[WAVES][64];
    Place places[PLACES];
};
enum { BEAM_NONE, BEAM_LIVE, BEAM_DONE };

// Candidate `place` of list (beam, part).
__device__ __forceinline__ Place candidate(const BeamArgs& a, const BeamShared& sh, size_t row,
    uint32_t beam, uint32_t part, uint32_t place)
{
    if (sh.kind[beam] == BEAM_NONE) {
        return {0, 0};
    }
    if (sh.kind[beam] == BEAM_DONE) {
        return part || place ? Place{0, 0} : place_of(sh.base[beam], beam, ~0u, 0);
    }
    const uint64_t key = a.keys[((row + beam) * a.parts + part) * a.c.keep + place];
    if (!key) {
        return {0, 0};
    }
    const uint32_t rank = (uint32_t)(key >> 32);
    const double x = rank_logit(rank);
    return place_of(sh.base[beam] + ((x - (double)sh.most[beam]) - sh.log_z[beam]), beam, rank,
        (uint32_t)~(uint32_t)key);
}

// The best places of `live` waves' falling lists, in the first wave; all waves call it.
__device__ __forceinline__ Place join_places(Place (&lists)[WAVES][64], Place p, uint32_t live,
    uint32_t wave, uint32_t lane)
{
#pragma unroll 1
    while (live > 1) {
        const uint32_t half = (live + 1) / 2;
        if (wave >= half && wave < live) {
            lists[wave][lane] = p;
        }
        __syncthreads();
        if (wave + half < live) {
            p = merge_places(p, lists[wave + half][63 - lane], lane);
        }
        live = half;
    }
    return p;
}

// grid (groups).
__global__ void __launch_bounds__(64 * WAVES)
k_beam_join(BeamArgs a)
{
    __shared__ BeamShared sh;
    const lh_beam_choice& c = a.c;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t group = blockIdx.x, row = group * c.beams;
    if (threadIdx.x == 0) {
        sh.bad = 0;
        sh.count = 0;
    }
    const uint32_t lists = c.beams * a.parts;
    __syncthreads();
    for (uint32_t b = wave; b < c.beams; b += WAVES) {
        const float s = c.scores[row + b];
        const bool live = scans(c, row + b);
        Range r = {0, 0, -__builtin_inff(), 0};
        if (live && lane < a.parts) {
            r = a.ranges[(row + b) * a.parts + lane];
        }
        rescale(r, wave_max64(r.m));
        r.z = wave_sum(r.z, lane);
        const bool odd = __ballot(r.bad != 0) != 0 || !(s < __builtin_inff());
        if (lane == 0) {
            sh.kind[b] = s == -__builtin_inff() ? BEAM_NONE : live ? BEAM_LIVE : BEAM_DONE;
            sh.base[b] = s;
            sh.most[b] = r.m;
            sh.log_z[b] = log(r.z);
            if (odd) {
                sh.bad = 1;
            }
        }
    }
    __syncthreads();
    if (sh.bad) {
        if (threadIdx.x < c.keep) {
            const size_t at = group * c.keep + threadIdx.x;
            c.parent[at] = -1;
            c.token[at] = -1;
            c.score[at] = __builtin_nanf("");
            if (c.done_out) {
                c.done_out[at] = 0;
            }
        }
        return;
    }
    Place p = {0, 0};
    uint32_t n = lists * c.keep;
    const bool few = n <= FEW;
    if (few) {
        // A candidate's place is the number of better ones, counted by the waves in shares:
        // the choice of 4 of 4 beams in both launches 11.7 us, sorted 13.4. The pairs of 256
        // candidates take longer (14.5) than their sorting.
        const uint32_t i = threadIdx.x % FEW, from = threadIdx.x / FEW * SHARE;
        if (threadIdx.x < FEW) {
            const uint32_t list = i / c.keep;
            sh.rank[i] = 0;
            sh.places[i] = i < n ? candidate(a, sh, row, list / a.parts, list % a.parts, i % c.keep)
                : Place{0, 0};
        } else if (wave == WAVES - 1) {
            sh.lists[0][lane] = {0, 0};
        }
        __syncthreads();
        const Place mine = sh.places[i];
        uint32_t better = 0;
#pragma unroll
        for (uint32_t j = 0; j < SHARE; j++) {
            better += sh.places[from + j] > mine;
        }
        atomicAdd(&sh.rank[i], better);
        __syncthreads();
        if (threadIdx.x < FEW && mine.score && sh.rank[i] < c.keep) {
            sh.lists[0][sh.rank[i]] = mine;
        }
        __syncthreads();
        p = sh.lists[0][lane];
    } else if (n <= 64 * WAVES) {
        // A candidate a thread.
        const uint32_t list = threadIdx.x / c.keep;
        if (threadIdx.x < n) {
            p = candidate(a, sh, row, list / a.parts, list % a.parts, threadIdx.x % c.keep);
        }
        p = sort_places(p, lane, true);
    } else {
        // Lists are falling, so the keep-th best of their first places bounds the group's best
        // from below, and only `keep` lists reach it. A list a lane of the first four waves:
        // a group has 256 at most (beam_parts).
        if (threadIdx.x < lists) {
            p = candidate(a, sh, row, threadIdx.x / a.parts, threadIdx.x % a.parts, 0);
        }
        p = sort_places(p, lane, true);
        p = join_places(sh.lists, p, (lists + 63) / 64, wave, lane);
        if (threadIdx.x == c.keep - 1) {
            sh.bound = p;
        }
        __syncthreads();
        const Place bound = sh.bound;
        for (uint32_t i = threadIdx.x; i < n; i += 64 * WAVES) {
            const uint32_t list = i / c.keep;
            const Place mine = candidate(a, sh, row, list / a.parts, list % a.parts, i % c.keep);
            if (mine.score && !(bound > mine)) {
                sh.places[atomicAdd(&sh.count, 1u)] = mine;
            }
        }
        __syncthreads();
        n = sh.count;
        p = {0, 0};
        for (uint32_t i = 64 * wave; i < n; i += 64 * WAVES) {
            const Place mine = i + lane < n ? sh.places[i + lane] : Place{0, 0};
            p = i < 64 * WAVES ? sort_places(mine, lane, true)
                : merge_places(p, sort_places(mine, lane, false), lane);
        }
    }
    if (!few) {
        p = join_places(sh.lists, p, (n + 63) / 64 < WAVES ? (n + 63) / 64 : WAVES, wave, lane);
    }
    if (threadIdx.x < c.keep) {
        const size_t at = group * c.keep + threadIdx.x;
        const bool any = p.score != 0;
        const uint32_t beam = 63 - (uint32_t)(p.rest >> 56);
        const bool ended = any && sh.kind[any ? beam : 0] == BEAM_DONE;
        const int64_t token = !any || ended ? -1
            : (int64_t)(0xffffffu - ((uint32_t)p.rest & 0xffffffu));
        c.parent[at] = any ? (int32_t)beam : -1;
        c.token[at] = token;
        c.score[at] = any ? (float)rank_score(p.score) : -__builtin_inff();
        if (c.done_out) {
            c.done_out[at] = ended || (token >= 0 && token == c.stop);
        }
    }
}

// ---- reordering ----

struct ReorderArgs {
    uint8_t* pages[LH_BEAM_LAYERS];
    const int32_t *parent, *length, *table;
    int32_t* table_out;
    size_t page_bytes;
    uint32_t layers, beams, width, page_size, page_count;
};

// What becomes of a group's beams, the same in every lane: of beam k (any lane may ask)
// its parent (-1: none) and the beam whose own pages it takes.
struct Family {
    int32_t parent;      // lane b: of beam b
    uint64_t keeps;      // children that take over their parent's own pages
    uint64_t dead;       // beams without children

    __device__ __forceinline__ Family(const int32_t* parents, uint32_t beams, uint32_t lane)
    {
        parent = lane < beams ? parents[lane] : -1;
        parent = parent >= 0 && (uint32_t)parent < beams ? parent : -1;
        uint64_t seen = 0;
        keeps = 0;
        for (uint32_t b = 0; b < beams; b++) {
            const int32_t p = __builtin_amdgcn_readlane(parent, b);
            if (p >= 0 && !(seen >> p & 1)) {
                keeps |= (uint64_t)1 << b;
                seen |= (uint64_t)1 << p;
            }
        }
        dead = ~seen & (beams == 64 ? ~(uint64_t)0 : ((uint64_t)1 << beams) - 1);
    }
    // The lane's own beam's.
    __device__ __forceinline__ uint32_t owner(uint32_t lane) const
    {
        if (keeps >> lane & 1) {
            return parent;
        }
        uint64_t left = dead;
        for (uint32_t turn = __popcll(~keeps & (((uint64_t)1 << lane) - 1)); turn && left; turn--) {
            left &= left - 1;
        }
        return left ? __builtin_ctzll(left) : lane;
    }
};

__device__ __forceinline__ uint32_t open_column(const ReorderArgs& a, int32_t length)
{
    return length < 0 ? 0 : (uint32_t)length / a.page_size;
}

// grid (pieces, sequences, layers and, for other tables than the old, one): the open pages
// that are copied, then the sequences' rows. No page is both read and written: the pages
// read stay their first child's, those written belong to beams without children.
// Bound: the pages' bytes; 8 groups of 8 beams in FP16 pages of 26 layers (436 MB
// both ways) 74 us, 5.9 TB/s; 4 beams in 4-bit pages 4.5 us, the loads of parents, length,
// page ids and page one after another.
__global__ void __launch_bounds__(256)
k_beam_copy(ReorderArgs a)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t group = blockIdx.y / a.beams, beam = blockIdx.y % a.beams;
    const size_t row = (size_t)group * a.beams;
    const int32_t length = a.length[row];
    const Family f(a.parent + row, a.beams, lane);
    const int32_t parent = __builtin_amdgcn_readlane(f.parent, beam);
    const uint32_t owner = __builtin_amdgcn_readlane(f.owner(lane), beam);
    const uint32_t column = open_column(a, length);
    if (blockIdx.z == a.layers) {
        const int32_t* full = a.table + (row + (parent < 0 ? owner : parent)) * a.width;
        const int32_t* own = a.table + (row + owner) * a.width;
        int32_t* out = a.table_out + (row + beam) * a.width;
        for (uint32_t c = blockIdx.x * 256 + threadIdx.x; c < a.width; c += gridDim.x * 256) {
            out[c] = (c < column ? full : own)[c];
        }
        return;
    }
    if (parent < 0 || f.keeps >> beam & 1 || length <= 0 || length % a.page_size == 0 ||
        column >= a.width) {
        return;
    }
    const int32_t from = a.table[(row + parent) * a.width + column];
    const int32_t to = a.table[(row + owner) * a.width + column];
    if (from < 0 || to < 0 || (uint32_t)from >= a.page_count || (uint32_t)to >= a.page_count) {
        return;
    }
    const uint4* source = reinterpret_cast<const uint4*>(a.pages[blockIdx.z] +
        from * a.page_bytes);
    uint4* target = reinterpret_cast<uint4*>(a.pages[blockIdx.z] + to * a.page_bytes);
    const size_t words = a.page_bytes / 16;
    for (size_t i = blockIdx.x * 256 + threadIdx.x; i < words; i += gridDim.x * 256) {
        target[i] = source[i];
    }
}

// grid (column tiles, groups): rows of tables in place. All of a group are read before one
// is written. A launch after the copies' takes 3.4 us (4 beams above 7.9 in all) to 5.3 (79).
__global__ void __launch_bounds__(256)
k_beam_tables(ReorderArgs a)
{
    __shared__ int32_t tile[LH_BEAMS][64];
    __shared__ int32_t from[LH_BEAMS], own[LH_BEAMS];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = (size_t)blockIdx.y * a.beams;
    const uint32_t column = open_column(a, a.length[row]);
    const Family f(a.parent + row, a.beams, lane);
    if (wave == 0) {
        const uint32_t owner = f.owner(lane);
        own[lane] = owner;
        from[lane] = f.parent < 0 ? owner : f.parent;
    }
    for (uint32_t first = blockIdx.x * 64; first < a.width; first += gridDim.x * 64) {
        const uint32_t at = first + lane;
        __syncthreads();
        for (uint32_t b = wave; b < a.beams; b += 4) {
            tile[b][lane] = at < a.width ? a.table[(row + b) * a.width + at] : 0;
        }
        __syncthreads();
        for (uint32_t b = wave; b < a.beams; b += 4) {
            if (at < a.width) {
                a.table_out[(row + b) * a.width + at] = tile[at < column ? from[b] : own[b]][lane];
            }
        }
    }
}

}  // namespace lh

using namespace lh;

// Workgroups of a row, as for log probabilities: one for each unit of the chip in all, each
// wave with a chunk at least. A group's beams have 256 together, or one each.
static uint32_t beam_parts(uint32_t rows, uint32_t vocab)
{
    const uint32_t chunks = (vocab + CHUNK - 1) / CHUNK, most = (chunks + WAVES - 1) / WAVES;
    uint32_t parts = 256 / rows;
    parts = parts < most ? parts : most;
    parts = parts ? parts : 1;
    return parts < 64 ? parts : 64;
}

extern "C" size_t lh_beam_scratch_bytes(uint32_t groups, uint32_t beams, uint32_t vocab,
    uint32_t keep)
{
    const size_t rows = (size_t)groups * beams, parts = beam_parts(rows, vocab);
    return lh_round16(rows * parts * (sizeof(Range) + 8 * (size_t)keep));
}

extern "C" int lh_launch_beam_select(const lh_beam_choice* choice, uint8_t* scratch,
    hipStream_t s)
{
    const uint32_t rows = choice->groups * choice->beams, parts = beam_parts(rows, choice->vocab);
    Range* ranges = reinterpret_cast<Range*>(scratch);
    const BeamArgs a = {*choice, ranges,
        reinterpret_cast<uint64_t*>(ranges + (size_t)rows * parts), parts};
    hipLaunchKernelGGL(k_beam_parts, dim3(parts, rows), dim3(64 * WAVES), 0, s, a);
    if (const hipError_t e = hipGetLastError()) {
        return (int)e;
    }
    hipLaunchKernelGGL(k_beam_join, dim3(choice->groups), dim3(64 * WAVES), 0, s, a);
    return (int)hipGetLastError();
}

extern "C" int lh_launch_beam_reorder(const lh_paged_cache* caches, uint32_t layers,
    uint32_t groups, uint32_t beams, const int32_t* parent, const int32_t* length,
    const int32_t* table, int32_t* table_out, uint32_t width, hipStream_t s)
{
    ReorderArgs a = {};
    for (uint32_t i = 0; i < layers; i++) {
        a.pages[i] = static_cast<uint8_t*>(caches[i].d_pages);
    }
    a.parent = parent, a.length = length, a.table = table, a.table_out = table_out;
    a.page_bytes = lh_paged_cache_bytes(caches) / caches->pages;
    a.layers = layers, a.beams = beams, a.width = width;
    a.page_size = caches->page_size, a.page_count = caches->pages;
    const uint32_t pieces = (uint32_t)((a.page_bytes + 16383) / 16384);
    hipLaunchKernelGGL(k_beam_copy, dim3(pieces, groups * beams, layers + (table != table_out)),
        dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e || table != table_out) {
        return (int)e;
    }
    const uint32_t tiles = (width + 63) / 64;
    hipLaunchKernelGGL(k_beam_tables, dim3(tiles < 256 ? tiles : 256, groups), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}
