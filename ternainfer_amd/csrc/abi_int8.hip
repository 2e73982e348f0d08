// C ABI of the matrix product in 8-bit integers (int8_linear_kernel.h).  Declarations: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "int8_linear_kernel.h"

using namespace terna;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool int8_rows_ok(int R, int K) { return R >= 1 && R <= 1 << 28 && K >= 1 && K <= kInt8MaxK; }

template <typename E>
void launch_quantise(const E* x, long long row, void* packed, float* scale, int R, int K, hipStream_t st)
{
    const int wide = aligned16(x) && (row * static_cast<long long>(sizeof(E)) & 15) == 0;
    uint8_t* const to = static_cast<uint8_t*>(packed);
    if (R < 2048) launch(terna_int8_quantise_kernel<E, 1>, dim3(R), dim3(kInt8Threads), 0, st, x, row, to, scale, R, K, wide);
    else launch(terna_int8_quantise_kernel<E, 16>, dim3((R + 15) / 16), dim3(kInt8Threads), 0, st, x, row, to, scale, R, K, wide);
}

template <typename Out, int WN, int WM, int NA, int MB, int SK, int ST>
bool launch_int8(Int8Linear a, hipStream_t st)
{
    using Tile = Int8Tile<WN, WM, NA, MB, SK, ST>;
    a.tiles_m = (a.M + Tile::BM - 1) / Tile::BM, a.tiles_n = (a.N + Tile::BN - 1) / Tile::BN;
    const long long grid = static_cast<long long>(a.tiles_m) * a.tiles_n;
    if (!launch_fits(grid, 256)) return false;
    auto kernel = terna_int8_linear_kernel<Out, WN, WM, NA, MB, SK, ST>;
    if (Tile::kBytes > kPlainLds) allow_dynamic_lds(kernel, Tile::kBytes, "hipFuncSetAttribute(int8 linear)", __LINE__);
    launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), Tile::kBytes, st, a);
    return true;
}
template <typename Out>
bool launch_int8_linear(const Int8Linear& a, hipStream_t st)
{
    if (a.M <= 32) return launch_int8<Out, 4, 1, 1, 1, 2, 4>(a, st);
    if (a.M <= 64) return launch_int8<Out, 4, 1, 1, 2, 1, 6>(a, st);
    if (a.M <= 512) return launch_int8<Out, 2, 2, 2, 2, 1, 5>(a, st);
    return launch_int8<Out, 2, 2, 4, 4, 1, 4>(a, st);
}

}  // namespace

extern "C" {

long long ternaspmm_int8_bytes(int R, int K) { return int8_rows_ok(R, K) ? int8_bands(R) * int8_k_blocks(K) * 1024 : -1; }

int ternaspmm_int8_quantise(const void* x, long long row, int fp32, void* packed, float* scale, int R, int K, terna_stream stream)
{
    if (!int8_rows_ok(R, K) || !x || !packed || !scale || !aligned16(packed) || (reinterpret_cast<uintptr_t>(x) & (fp32 ? 3 : 1)) || row < 0 || !launch_fits(R, kInt8Threads / 16))
        return -1;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (fp32) launch_quantise(static_cast<const float*>(x), row, packed, scale, R, K, st);
    else launch_quantise(static_cast<const uint16_t*>(x), row, packed, scale, R, K, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_int8_quantise", e, __LINE__);
    return 0;
}

int ternaspmm_int8_pack(const void* x, long long row, void* packed, int R, int K, terna_stream stream)
{
    if (!int8_rows_ok(R, K) || !x || !packed || !aligned16(packed) || row < 0 || !launch_fits((R + 15) / 16, kInt8Threads)) return -1;
    launch(terna_int8_pack_kernel, dim3((R + 15) / 16), dim3(kInt8Threads), 0, static_cast<hipStream_t>(stream), static_cast<const uint8_t*>(x), row,
           static_cast<uint8_t*>(packed), R, K, aligned16(x) && (row & 15) == 0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_int8_pack", e, __LINE__);
    return 0;
}

int ternaspmm_int8_linear(const void* x, const float* x_scale, const void* w, const float* w_scale, void* out, int fp32, int M, int N, int K, terna_stream stream)
{
    if (!int8_rows_ok(M, K) || !int8_rows_ok(N, K) || !x || !x_scale || !w || !w_scale || !out || !aligned16(x) || !aligned16(w) || !aligned16(out)) return -1;
    Int8Linear a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), x_scale, w_scale, out, M, N, K, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!(fp32 ? launch_int8_linear<float>(a, st) : launch_int8_linear<uint16_t>(a, st))) return -1;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_int8_linear", e, __LINE__);
    return 0;
}

}  // extern "C"
