// C ABI of rotary positions (rotary_kernel.h).  Declaration: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "rotary_kernel.h"

using namespace terna;

namespace {

template <typename T, bool ADJACENT>
void launch_rotary(const void* x, void* out, const long long* pos, const double* frequency, const RotaryRows& in, const RotaryRows& to, const RotaryShape& s, int in_place,
                   bool pieces, dim3 grid, hipStream_t st)
{
    launch(pieces ? terna_rotary_kernel<T, ADJACENT> : terna_rotary_pairs_kernel<T, ADJACENT>, grid, dim3(kRotaryThreads), 0, st, static_cast<const T*>(x),
           static_cast<T*>(out), pos, frequency, in, to, s, in_place);
}

}  // namespace

extern "C" {

int ternaspmm_rotary(const void* x, const long long* x_strides, void* out, const long long* out_strides, int fp32, const long long* pos, int per_sequence,
                     const double* frequency, int pairs, double amplitude, int B, int T, int H, int D, int adjacent, terna_stream stream)
{
    if (!x || !out || !x_strides || !out_strides || !pos || !frequency || B < 1 || T < 1 || H < 1 || D < 2 || D > 1024 || pairs < 1 || 2 * pairs > D ||
        H > 65535 || static_cast<long long>(B) * T > 1 << 30)
        return -1;
    const RotaryRows in{x_strides[0], x_strides[1], x_strides[2]}, to{out_strides[0], out_strides[1], out_strides[2]};
    const int size = fp32 ? 4 : 2, n = 16 / size;
    const bool in_place = x == out;
    if (in_place && (in.batch != to.batch || in.token != to.token || in.head != to.head)) return -1;
    auto whole = [&](const void* p, const RotaryRows& r) { return ((reinterpret_cast<uintptr_t>(p) & 15) | ((r.batch | r.token | r.head) & (n - 1))) == 0; };
    const bool pieces = D % n == 0 && whole(x, in) && whole(out, to) && (adjacent || pairs % n == 0);
    RotaryShape s{T, H, D, pairs, per_sequence != 0, B * T, 1, amplitude};
    // Tokens a workgroup: as many as its angles have room for while a thread has no more than four pieces (us, 32768 tokens of one head of 128 dimensions in
    // bf16: one token 25.5, so 10.5; of 25 heads, where this is one: 74.9, four 81.8).  Where that leaves CUs without a workgroup, the heads of a token
    // go to several (one token of 200 heads 8.6, so 3.5).
    const long long steps = static_cast<long long>(H) * (pieces ? D / n : D - pairs);
    while (2 * s.tokens_a_group * pairs <= kRotaryMaxAngles && 2 * s.tokens_a_group * steps <= 4 * kRotaryThreads && s.tokens / (2 * s.tokens_a_group) >= 512 &&
           (T == 1 || 2 * s.tokens_a_group <= T))
        s.tokens_a_group *= 2;
    const int groups = (s.tokens + s.tokens_a_group - 1) / s.tokens_a_group;
    if (!launch_fits(groups, kRotaryThreads)) return -1;
    int slices = 1;
    while (slices < 64 && groups * slices < 512 && 2 * slices * kRotaryThreads <= s.tokens_a_group * steps) slices *= 2;
    const dim3 grid(groups, slices);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (fp32 && adjacent) launch_rotary<float, true>(x, out, pos, frequency, in, to, s, in_place, pieces, grid, st);
    else if (fp32) launch_rotary<float, false>(x, out, pos, frequency, in, to, s, in_place, pieces, grid, st);
    else if (adjacent) launch_rotary<uint16_t, true>(x, out, pos, frequency, in, to, s, in_place, pieces, grid, st);
    else launch_rotary<uint16_t, false>(x, out, pos, frequency, in, to, s, in_place, pieces, grid, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_rotary", e, __LINE__);
    return 0;
}

}  // extern "C"
