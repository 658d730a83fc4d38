// Beam search: the selection of hypotheses and the reordering of their states.
#include <algorithm>
#include <cmath>
#include <numeric>
#include <vector>

#include "decode_common.h"

namespace leo {
namespace {

constexpr uint32_t kMostBeams = 64;

__device__ __forceinline__ float negative_infinity() { return -__builtin_inff(); }

// Floats in the order of whole numbers, -inf above 0.
__device__ __forceinline__ uint32_t order_key(float z) {
    const uint32_t b = __float_as_uint(z);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A symbol of a row as one number: the larger logit first, of equals the lower
// symbol. 0 is none.
__device__ __forceinline__ uint64_t candidate(float z, uint32_t at) {
    return static_cast<uint64_t>(order_key(z + 0.0f)) << 32 | (0xffffffffu - at);
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    for (int step = 32; step; step /= 2) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(v), step);
        v = other > v ? other : v;
    }
    return v;
}

// What a row leaves for its search: its log of the sum of exponentials above its
// largest logit, and its `kept` best candidates in falling order.
struct BeamRecord {
    float top;
    uint32_t pad0;
    double log_sum;
};

__device__ __forceinline__ bool is_finished(const LeoBeams& a, uint64_t row) { return a.finished && a.finished[row]; }

// One workgroup a row.
template <class T>
__global__ __launch_bounds__(256) void leo_beam_rows(LeoBeams a, BeamRecord* records, uint64_t* candidates) {
    __shared__ float tops[4];
    __shared__ double sums[4];
    __shared__ uint64_t bests[4];
    const uint64_t row = blockIdx.x;
    const uint32_t n = static_cast<uint32_t>(a.symbols), lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    if (is_finished(a, row) || !(a.scores[row] > negative_infinity())) return;
    const auto* logits = static_cast<const typename T::type*>(a.logits) + row * a.logits_stride;
    float top = negative_infinity();
    for (uint32_t v = threadIdx.x; v < n; v += 256) top = fmaxf(top, T::load(logits, v));
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0.0;
    for (uint32_t v = threadIdx.x; v < n; v += 256) {
        const float z = T::load(logits, v);
        sum += z == top ? 1.0 : z > negative_infinity() ? exp(static_cast<double>(z) - top) : 0.0;
    }
    for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) records[row] = {top, 0, log(sums[0] + sums[1] + sums[2] + sums[3])};
    uint64_t below = ~0ull;
    for (uint32_t k = 0; k < a.kept; ++k) {
        uint64_t best = 0;
        if (below)
            for (uint32_t v = threadIdx.x; v < n; v += 256) {
                const float z = T::load(logits, v);
                const uint64_t c = z > negative_infinity() ? candidate(z, v) : 0;
                if (c < below && c > best) best = c;
            }
        best = wave_max64(best);
        __syncthreads();
        if (lane == 0) bests[wave] = best;
        __syncthreads();
        for (uint32_t w = 0; w < 4; ++w) best = bests[w] > best ? bests[w] : best;
        if (threadIdx.x == 0) candidates[row * a.kept + k] = best;
        below = best;
    }
}

struct Ranked {
    double rank;
    uint32_t at;  // hypothesis * kept + place in its row's order
};
__device__ __forceinline__ bool before(const Ranked& p, const Ranked& q) { return p.rank > q.rank || (p.rank == q.rank && p.at < q.at); }

// One wave a search.
__global__ __launch_bounds__(64) void leo_beam_groups(LeoBeams a, const BeamRecord* records, const uint64_t* candidates) {
    const uint64_t group = blockIdx.x, first = group * a.beams;
    const uint32_t lane = threadIdx.x, kept = static_cast<uint32_t>(a.kept), count = static_cast<uint32_t>(a.beams) * kept;
    const auto length_of = [&](uint64_t row) {
        return a.lengths ? static_cast<int64_t>(a.lengths[row]) + (is_finished(a, row) ? 0 : 1) : 1;
    };
    const auto score_of = [&](uint32_t at) -> double {  // -inf where there is none
        const uint64_t row = first + at / kept;
        const float score = a.scores[row];
        if (!(score > negative_infinity())) return -__builtin_inf();
        if (is_finished(a, row)) return at % kept == 0 ? static_cast<double>(score) : -__builtin_inf();
        const uint64_t c = candidates[row * kept + at % kept];
        if (c == 0) return -__builtin_inf();
        const float z = from_order_key(static_cast<uint32_t>(c >> 32));
        return score + ((z == records[row].top ? 0.0 : static_cast<double>(z) - records[row].top) - records[row].log_sum);
    };
    Ranked last = {__builtin_inf(), 0};
    bool any = false;  // `last` was taken
    for (uint32_t k = 0; k < kept; ++k) {
        Ranked best = {-__builtin_inf(), 0xffffffffu};
        for (uint32_t at = lane; at < count; at += 64) {
            const double score = score_of(at);
            if (!(score > -__builtin_inf())) continue;
            const int64_t length = length_of(first + at / kept);
            const double norm = a.length_penalty == 0.0 ? 1.0 : pow(static_cast<double>(length < 1 ? 1 : length), a.length_penalty);
            const Ranked mine = {score / norm, at};
            if ((!any || before(last, mine)) && (best.at == 0xffffffffu || before(mine, best))) best = mine;
        }
        for (int step = 32; step; step /= 2) {
            const Ranked other = {__shfl_xor(best.rank, step), static_cast<uint32_t>(__shfl_xor(static_cast<int>(best.at), step))};
            if (other.at != 0xffffffffu && (best.at == 0xffffffffu || before(other, best))) best = other;
        }
        const bool found = best.at != 0xffffffffu;
        if (lane == 0) {
            const uint64_t to = group * kept + k;
            const uint32_t beam = found ? best.at / kept : 0;
            const uint64_t row = first + beam;
            const bool was = found && is_finished(a, row);
            const uint32_t symbol = found && !was ? 0xffffffffu - static_cast<uint32_t>(candidates[row * kept + best.at % kept]) : 0xffffffffu;
            a.out_symbols[to] = static_cast<int32_t>(symbol);
            a.out_parents[to] = static_cast<int32_t>(beam);
            a.out_scores[to] = found ? static_cast<float>(score_of(best.at)) : negative_infinity();
            if (a.out_finished) a.out_finished[to] = was || (found && !was && static_cast<int64_t>(symbol) == a.end);
            if (a.out_lengths) a.out_lengths[to] = a.lengths[row] + (found && !was ? 1 : 0);
        }
        if (!found) {
            for (uint32_t j = k + 1 + lane; j < kept; j += 64) {
                const uint64_t to = group * kept + j;
                a.out_symbols[to] = -1;
                a.out_parents[to] = 0;
                a.out_scores[to] = negative_infinity();
                if (a.out_finished) a.out_finished[to] = 0;
                if (a.out_lengths) a.out_lengths[to] = a.lengths[first];
            }
            return;
        }
        last = best;
        any = true;
    }
}

struct BeamPlan {
    uint64_t candidates, workspace;  // the candidates' offset, and the whole
};
BeamPlan beam_plan(uint64_t groups, uint64_t beams, uint64_t kept) {
    const uint64_t rows = groups * beams;
    BeamPlan p{};
    p.candidates = (rows * sizeof(BeamRecord) + 255) / 256 * 256;
    p.workspace = p.candidates + rows * kept * sizeof(uint64_t);
    return p;
}

void check_beams(const char* who, uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols) {
    const auto need = [&](bool ok, const char* what) {
        if (!ok) throw Error(LEO_ERR_INVALID_ARGUMENT, std::string(who) + ": " + what);
    };
    need(beams >= 1 && beams <= kMostBeams, "beams must be 1 .. 64");
    need(kept >= 1 && kept <= kMostBeams, "kept must be 1 .. 64");
    need(groups <= 65535, "too many groups");
    need(symbols >= 1 && symbols <= 0x7fffffffu, "symbols must be 1 .. 2^31 - 1");
}

template <class T>
void launch_beams(const BeamPlan& p, const LeoBeams& b, hipStream_t stream) {
    auto* records = static_cast<BeamRecord*>(b.workspace);
    auto* candidates = reinterpret_cast<uint64_t*>(static_cast<char*>(b.workspace) + p.candidates);
    launch(leo_beam_rows<T>, dim3(static_cast<uint32_t>(b.groups * b.beams)), dim3(256), 0, stream, b, records, candidates);
    launch(leo_beam_groups, dim3(static_cast<uint32_t>(b.groups)), dim3(64), 0, stream, b, static_cast<const BeamRecord*>(records),
           static_cast<const uint64_t*>(candidates));
}

// --- reordering ------------------------------------------------------------------------------------------------------

// One workgroup 16 bytes a thread of one place of a row, for all of a search's
// targets: in place a thread holds what it moves in a column of LDS that is its
// own, so nothing waits for other threads.
constexpr uint32_t kArrays = 32;

struct ReorderArgs {
    LeoStateArray arrays[kArrays];
    uint64_t before[kArrays];  // workgroups of the arrays before
    uint32_t count;
    uint32_t groups, beams, kept;
    const int32_t* parents;
};

template <bool kInPlace>
__global__ __launch_bounds__(256) void leo_reorder(ReorderArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint4v held[];
    uint32_t which = 0;
    while (which + 1 < a.count && blockIdx.x >= a.before[which + 1]) ++which;
    const LeoStateArray& s = a.arrays[which];
    const uint64_t unit = blockIdx.x - a.before[which], wide = blockDim.x * 16, pieces = (s.width + wide - 1) / wide;
    const uint64_t piece = unit % pieces, outer = unit / pieces % s.outer, group = unit / pieces / s.outer;
    const uint64_t at = piece * wide + threadIdx.x * 16;
    if (at >= s.width) return;
    const uint32_t bytes = static_cast<uint32_t>(min<uint64_t>(16, s.width - at));
    const char* source = static_cast<const char*>(s.source) + outer * s.source_outer + at;
    char* target = static_cast<char*>(s.target) + outer * s.target_outer + at;
    const int32_t* parents = a.parents + group * a.kept;
    const auto read = [&](uint32_t k) {
        const int32_t parent = parents[k];
        uint4v v = {0, 0, 0, 0};
        if (parent < 0 || parent >= static_cast<int32_t>(a.beams)) return v;
        const char* from = source + static_cast<int64_t>(group * a.beams + parent) * s.source_row;
        if (bytes == 16) return load_16(from);
        for (uint32_t i = 0; i < bytes; ++i) v[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(from[i])) << (8 * (i % 4));
        return v;
    };
    const auto write = [&](uint32_t k, const uint4v& v) {
        char* to = target + static_cast<int64_t>(group * a.kept + k) * s.target_row;
        if (bytes == 16) {
            __builtin_memcpy(to, &v, 16);
            return;
        }
        for (uint32_t i = 0; i < bytes; ++i) to[i] = static_cast<char>(v[i / 4] >> (8 * (i % 4)));
    };
    if constexpr (kInPlace) {
        for (uint32_t k = 0; k < a.kept; ++k)
            if (parents[k] != static_cast<int32_t>(k)) held[k * blockDim.x + threadIdx.x] = read(k);
        for (uint32_t k = 0; k < a.kept; ++k)
            if (parents[k] != static_cast<int32_t>(k)) write(k, held[k * blockDim.x + threadIdx.x]);
    } else {
        for (uint32_t k = 0; k < a.kept; ++k) write(k, read(k));
    }
}

// The bytes from an array's first to its last.
struct Extent {
    uint64_t begin, end;
    uint32_t array;
    bool target;
};

// Whether a target shares a byte with another of them; sorts them.
bool any_meet(std::vector<Extent>& extents) {
    std::sort(extents.begin(), extents.end(), [](const Extent& p, const Extent& q) { return p.begin < q.begin; });
    uint64_t all = 0, targets = 0;  // the ends of what came before
    for (const Extent& e : extents) {
        if (e.begin < targets || (e.target && e.begin < all)) return true;
        all = std::max(all, e.end);
        if (e.target) targets = std::max(targets, e.end);
    }
    return false;
}

// The same for arrays whose ranges meet, as the columns of one buffer do: where the
// starts of all their rows (or of all pieces of them) lie apart modulo a common
// divisor of the strides, no two meet.
bool may_meet(const LeoReorder& r, const std::vector<Extent>& extents) {
    for (const bool pieces : {false, true}) {
        uint64_t modulus = 0;
        const auto strides_of = [&](const Extent& e, uint64_t& row, uint64_t& outer) {
            const LeoStateArray& s = r.arrays[e.array];
            const uint64_t rows = r.groups * (e.target ? r.kept : r.beams);
            row = rows == 1 ? 0 : static_cast<uint64_t>(e.target ? s.target_row : s.source_row);
            outer = s.outer == 1 ? 0 : static_cast<uint64_t>(e.target ? s.target_outer : s.source_outer);
        };
        uint64_t row, outer;
        for (const Extent& e : extents) {
            strides_of(e, row, outer);
            modulus = std::gcd(modulus, row);
            if (pieces) modulus = std::gcd(modulus, outer);
        }
        if (modulus == 0) return true;
        std::vector<Extent> folded;
        bool fits = true;
        for (const Extent& e : extents) {
            strides_of(e, row, outer);
            const LeoStateArray& s = r.arrays[e.array];
            const uint64_t length = s.width + (pieces ? 0 : (s.outer - 1) * outer), begin = e.begin % modulus;
            fits = fits && length <= modulus;
            folded.push_back({begin, std::min(begin + length, modulus), e.array, e.target});
            if (begin + length > modulus) folded.push_back({0, begin + length - modulus, e.array, e.target});
        }
        if (fits && !any_meet(folded)) return false;
    }
    return true;
}

// Refuses targets that share memory with anything else.
void check_apart(const LeoReorder& r, std::vector<Extent>& extents) {
    if (!any_meet(extents)) return;
    for (size_t from = 0; from < extents.size();) {
        std::vector<Extent> cluster;
        uint64_t end = 0;
        for (; from < extents.size() && (cluster.empty() || extents[from].begin < end); ++from) {
            end = std::max(end, extents[from].end);
            cluster.push_back(extents[from]);
        }
        std::vector<Extent> copy = cluster;
        require(!any_meet(copy) || !may_meet(r, cluster), "leo_reorder_states: a target overlaps another array");
    }
}

}  // namespace
}  // namespace leo

using namespace leo;

extern "C" {

int32_t leo_beam_workspace_bytes(uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols, uint64_t* bytes) {
    return guarded([&] {
        require(bytes, "leo_beam_workspace_bytes: null argument");
        check_beams("leo_beam_workspace_bytes", groups, beams, kept, symbols);
        *bytes = groups ? beam_plan(groups, beams, kept).workspace : 0;
    });
}

int32_t leo_beam_select(const LeoBeams* beams, void* stream) {
    return guarded([&] {
        require(beams, "leo_beam_select: null argument");
        const LeoBeams& b = *beams;
        check_beams("leo_beam_select", b.groups, b.beams, b.kept, b.symbols);
        require(valid_type(b.type), "leo_beam_select: unknown type");
        if (b.groups == 0) return;
        require(b.logits && b.scores && b.out_symbols && b.out_parents && b.out_scores, "leo_beam_select: null argument");
        require(b.logits_stride >= 0, "leo_beam_select: logits_stride must not be negative");
        require(std::isfinite(b.length_penalty), "leo_beam_select: length_penalty must be finite");
        require(b.lengths || (b.length_penalty == 0.0 && !b.out_lengths), "leo_beam_select: length_penalty or out_lengths without lengths");
        require(b.end >= -1 && b.end < static_cast<int64_t>(b.symbols), "leo_beam_select: end must be a symbol, or -1");
        const BeamPlan p = beam_plan(b.groups, b.beams, b.kept);
        require(b.workspace && reinterpret_cast<uintptr_t>(b.workspace) % 256 == 0 && b.workspace_bytes >= p.workspace,
                "leo_beam_select: workspace is missing, too small or not 256-byte aligned");
        const auto at = static_cast<hipStream_t>(stream);
        if (b.type == LEO_TYPE_F32) launch_beams<F32>(p, b, at);
        else if (b.type == LEO_TYPE_F16) launch_beams<F16>(p, b, at);
        else launch_beams<BF16>(p, b, at);
    });
}

int32_t leo_reorder_states(const LeoReorder* reorder, void* stream) {
    return guarded([&] {
        require(reorder, "leo_reorder_states: null argument");
        const LeoReorder& r = *reorder;
        require(r.beams >= 1 && r.beams <= kMostBeams, "leo_reorder_states: beams must be 1 .. 64");
        require(r.kept >= 1 && r.kept <= kMostBeams, "leo_reorder_states: kept must be 1 .. 64");
        require(r.groups <= 65535, "leo_reorder_states: too many groups");
        if (r.count == 0 || r.groups == 0) return;
        require(r.arrays && r.parents, "leo_reorder_states: null argument");
        require(r.count <= 65535, "leo_reorder_states: too many arrays");
        const uint64_t from_rows = r.groups * r.beams, to_rows = r.groups * r.kept;
        constexpr uint64_t kMost = 1ull << 46;  // of sizes and strides, so that their products stay inside 64 bits
        std::vector<Extent> extents;
        std::vector<uint32_t> order[2];  // arrays out of place, in place
        for (uint32_t i = 0; i < r.count; ++i) {
            const LeoStateArray& s = r.arrays[i];
            if (s.outer == 0 || s.width == 0) continue;
            require(s.source && s.target, "leo_reorder_states: null array");
            require(s.outer <= 0x7fffffffu && s.width <= kMost, "leo_reorder_states: an array is too large");
            for (int64_t stride : {s.source_row, s.source_outer, s.target_row, s.target_outer})
                require(stride >= 0 && static_cast<uint64_t>(stride) <= kMost, "leo_reorder_states: strides must be 0 .. 2^46");
            const auto span = [&](uint64_t rows, int64_t row, int64_t outer) {
                return static_cast<uint64_t>(static_cast<unsigned __int128>(rows - 1) * row + static_cast<unsigned __int128>(s.outer - 1) * outer) + s.width;
            };
            // each of a target's pieces has bytes of its own: rows of pieces, or pieces of rows
            const uint64_t row = static_cast<uint64_t>(s.target_row), outer = static_cast<uint64_t>(s.target_outer);
            const bool by_row = (s.outer == 1 || outer >= s.width) && (to_rows == 1 || row >= (s.outer - 1) * outer + s.width);
            const bool by_outer = (to_rows == 1 || row >= s.width) && (s.outer == 1 || outer >= (to_rows - 1) * row + s.width);
            require(by_row || by_outer, "leo_reorder_states: a target's rows overlap");
            const bool same = s.source == s.target;
            if (same)
                require(r.beams == r.kept && s.source_row == s.target_row && (s.outer == 1 || s.source_outer == s.target_outer),
                        "leo_reorder_states: an array that is its own target needs the same strides and as many kept as beams");
            order[same].push_back(i);
            const uintptr_t from = reinterpret_cast<uintptr_t>(s.source), to = reinterpret_cast<uintptr_t>(s.target);
            if (!same) extents.push_back({from, from + span(from_rows, s.source_row, s.source_outer), i, false});
            extents.push_back({to, to + span(to_rows, s.target_row, s.target_outer), i, true});
        }
        check_apart(r, extents);
        // in place, the rows of a piece are held in LDS: 64 KB
        const uint32_t threads = r.kept <= 16 ? 256 : 64;
        ReorderArgs a{};
        a.groups = static_cast<uint32_t>(r.groups);
        a.beams = static_cast<uint32_t>(r.beams);
        a.kept = static_cast<uint32_t>(r.kept);
        a.parents = r.parents;
        for (int in_place = 0; in_place < 2; ++in_place) {
            for (size_t from = 0; from < order[in_place].size();) {
                uint64_t units = 0;
                a.count = 0;
                for (; from < order[in_place].size() && a.count < kArrays; ++from) {
                    const LeoStateArray& s = r.arrays[order[in_place][from]];
                    const unsigned __int128 mine = static_cast<unsigned __int128>((s.width + threads * 16 - 1) / (threads * 16)) * s.outer * r.groups;
                    require(mine <= 0x7fffffffu, "leo_reorder_states: an array is too large");
                    if (units + static_cast<uint64_t>(mine) > 0x7fffffffu) break;
                    a.arrays[a.count] = s;
                    a.before[a.count++] = units;
                    units += static_cast<uint64_t>(mine);
                }
                const auto at = static_cast<hipStream_t>(stream);
                const dim3 grid(static_cast<uint32_t>(units)), block(threads);
                if (in_place) launch(leo_reorder<true>, grid, block, a.kept * threads * 16, at, a);
                else launch(leo_reorder<false>, grid, block, 0, at, a);
            }
        }
    });
}

}  // extern "C"
