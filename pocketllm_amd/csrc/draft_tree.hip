// The path of a drafted tree that the sampled tokens follow.  Node 0 holds the sequence's last token; node i's sampled token is what the model continues its path with.
// From node 0 on: the first child (its parent is the path's last node) whose drafted token is the one sampled there, until there is none.  Every node of
// the path but the first is a token that the model would have given by itself, and the token sampled at its last node is one more.
//
// A wave per sequence, four nodes to a lane, in registers: a step is a comparison, a ballot and three reads of a lane.  Bound: the chain of loads in front of that.
#include "paged_cache.h"
#include "pllm_internal.h"

namespace pllm {
namespace {

struct AcceptArgs {
    const int32_t* parents; const int64_t* drafted; const int64_t* sampled; const int32_t* lengths; const int32_t* cu_steps;
    int32_t* kept; int32_t* counts; int64_t* tokens; int32_t* new_lengths;
    int rows, seqs, even, most;
};

__device__ __forceinline__ int64_t read_lane(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32), lane);
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

__global__ __launch_bounds__(64) void draft_tree_accept_kernel(const AcceptArgs a) {
    constexpr int kPer = kTreeNodes / 64;
    const int s = blockIdx.x, lane = threadIdx.x;
    const int offset = paged_offset(a.cu_steps, s, a.even, a.rows), n = paged_offset(a.cu_steps, s + 1, a.even, a.rows) - offset;
    const int nodes = min(max(n, 0), kTreeNodes);
    int parent[kPer];
    int64_t drafted[kPer], sampled[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int node = 64 * i + lane, at = offset + node;
        const bool there = node < nodes;
        parent[i] = there ? a.parents[at] : -1;
        drafted[i] = there ? a.drafted[at] : 0;
        sampled[i] = there ? a.sampled[at] : 0;
    }
    int32_t* kept = a.kept + static_cast<size_t>(s) * a.most;
    int here = 0, count = nodes > 0 ? 1 : 0, mine = -1;                       // mine: the path's node of number 64 c + lane, c the stretch being walked
    int64_t token = nodes > 0 ? read_lane(sampled[0], 0) : -1;
    if (lane == 0 && count) mine = 0;
    while (count > 0 && count < a.most) {
        int next = -1;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int node = 64 * i + lane;
            const uint64_t follows = __ballot(node > here && node < nodes && parent[i] == here && drafted[i] == token);
            if (next < 0 && follows) next = 64 * i + __ffsll(static_cast<unsigned long long>(follows)) - 1;
        }
        if (next < 0) break;
        if (count % 64 == 0) {
            kept[count - 64 + lane] = mine;
            mine = -1;
        }
        here = __builtin_amdgcn_readfirstlane(next);
        if (lane == count % 64) mine = here;
        ++count;
        const int from = here & 63;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (here >> 6 == i) token = read_lane(sampled[i], from);
    }
    const int stretch = count > 0 ? (count - 1) / 64 * 64 : 0;
    if (stretch + lane < a.most) kept[stretch + lane] = mine;
    for (int i = stretch + 64 + lane; i < a.most; i += 64) kept[i] = -1;
    if (lane == 0) {
        a.counts[s] = count;
        a.tokens[s] = token;
        const int64_t length = static_cast<int64_t>(a.lengths[s]) - n + count;
        a.new_lengths[s] = static_cast<int>(length < 0 ? 0 : length);
    }
}

}  // namespace
}  // namespace pllm

extern "C" int pllm_draft_tree_accept(const int32_t* parents, const int64_t* drafted, const int64_t* sampled, const int32_t* lengths, const int32_t* cu_steps, int64_t rows, int64_t seqs,
                                      int64_t most, int32_t* kept, int32_t* counts, int64_t* tokens, int32_t* new_lengths, void* stream) {
    using namespace pllm;
    if (!parents || !drafted || !sampled || !lengths || !kept || !counts || !tokens || !new_lengths || rows <= 0 || seqs <= 0 || most <= 0) return PLLM_ERR_INVALID_ARGUMENT;
    if (!cu_steps && rows % seqs != 0) return PLLM_ERR_INVALID_ARGUMENT;
    if (rows > 0x3fffff || seqs > 0xfffff || most > kTreeNodes || (!cu_steps && rows / seqs > kTreeNodes)) return PLLM_ERR_UNSUPPORTED;
    const uintptr_t words = reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(cu_steps) | reinterpret_cast<uintptr_t>(kept) |
                            reinterpret_cast<uintptr_t>(counts) | reinterpret_cast<uintptr_t>(new_lengths);
    const uintptr_t doubles = reinterpret_cast<uintptr_t>(drafted) | reinterpret_cast<uintptr_t>(sampled) | reinterpret_cast<uintptr_t>(tokens);
    if ((words & 3u) || (doubles & 7u)) return PLLM_ERR_INVALID_ARGUMENT;
    AcceptArgs a{parents, drafted, sampled, lengths, cu_steps, kept, counts, tokens, new_lengths, static_cast<int>(rows), static_cast<int>(seqs),
                 cu_steps ? 0 : static_cast<int>(rows / seqs), static_cast<int>(most)};
    hipLaunchKernelGGL(draft_tree_accept_kernel, dim3(static_cast<unsigned>(seqs)), dim3(64), 0, static_cast<hipStream_t>(stream), a);
    return hipGetLastError() == hipSuccess ? PLLM_OK : PLLM_ERR_LAUNCH;
}
