// C ABI of the log probabilities of given tokens (logprobs_kernel.h).  Declarations: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "logprobs_kernel.h"

using namespace terna;

namespace {

bool logprobs_shape_ok(int M, int V, int top)
{
    return M >= 1 && M <= 1 << 24 && V >= 1 && V <= 1 << 22 && top >= 0 && top <= kLogprobMaxTop && top <= V;
}

// Workgroups of a row: no more blocks each than LDS has room for, and enough that the rows together give every CU two, while each keeps two pieces a thread
// and the merge's keys fit its LDS.
int logprobs_least_splits(int V, int fp32)
{
    const int pieces = V / (fp32 ? 4 : 8) + 2, most = 16 * kLogprobBlocks;
    return (pieces + most - 1) / most;
}
int logprobs_splits(int M, int V, int top, int fp32)
{
    int splits = logprobs_least_splits(V, fp32);
    while (2 * splits <= kLogprobThreads && M * splits < 512 && V / (2 * splits) >= 4 * 2 * kLogprobThreads && 2 * splits * top <= kLogprobKeys) splits *= 2;
    return splits;
}

}  // namespace

extern "C" {

long long ternaspmm_token_logprobs_workspace_bytes(int M, int V, int fp32, int top)
{
    if (!logprobs_shape_ok(M, V, top)) return -1;
    const int splits = logprobs_splits(M, V, top, fp32);
    return splits == 1 ? 0 : static_cast<long long>(M) * splits * (8ll * top + static_cast<long long>(sizeof(LogprobStats)));
}

int ternaspmm_token_logprobs(const void* logits, long long row, int fp32, const long long* targets, float* logprob, float* entropy, long long* top_ids,
                             float* top_logprobs, int top, void* workspace, int M, int V, terna_stream stream)
{
    if (!logprobs_shape_ok(M, V, top) || !logits || !entropy || (targets && !logprob) || (top && (!top_ids || !top_logprobs)) ||
        (reinterpret_cast<uintptr_t>(workspace) & 7) || (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)) || row < 0)
        return -1;
    LogprobArgs a{logits, targets, logprob, entropy, top_ids, top_logprobs, workspace, row, M, V, top, workspace ? logprobs_splits(M, V, top, fp32) : 1};
    if (a.splits < logprobs_least_splits(V, fp32)) return -1;
    const long long grid = static_cast<long long>(M) * a.splits;
    if (grid >= 1ll << 31) return -1;
    hipStream_t st = static_cast<hipStream_t>(stream);
    launch(fp32 ? terna_logprobs_kernel<float> : terna_logprobs_kernel<uint16_t>, dim3(static_cast<unsigned>(grid)), dim3(kLogprobThreads), 0, st, a);
    if (a.splits > 1) launch(fp32 ? terna_logprobs_merge_kernel<float> : terna_logprobs_merge_kernel<uint16_t>, dim3(M), dim3(kLogprobThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_token_logprobs", e, __LINE__);
    return 0;
}

}  // extern "C"
