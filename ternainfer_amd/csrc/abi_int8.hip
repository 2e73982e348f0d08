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
    const int held = (4 * int8_k_blocks(K) + 63) / 64;
    auto kernel = held <= 1 ? terna_int8_quantise_kernel<E, 1> : held <= 3 ? terna_int8_quantise_kernel<E, 3> : terna_int8_quantise_kernel<E, 7>;
    launch(kernel, dim3(static_cast<unsigned>((R + 31ll) / 32 * 8)), dim3(kInt8Threads), 0, st, x, row, to, scale, R, K, wide);
}

template <typename Out, int KIND, int WN, int WM, int NA, int MB, int SK, int ST>
void launch_int8(const Int8Linear& a, long long tiles, hipStream_t st)
{
    using Tile = Int8Tile<WN, WM, NA, MB, SK, ST>;
    static_assert(Tile::BN == kInt8Tiles[KIND].features && Tile::BM == kInt8Tiles[KIND].rows);
    constexpr int lds = Tile::template bytes<Out>(), join_lds = 32 * WM * Tile::template pitch<Out>();
    auto kernel = terna_int8_linear_kernel<Out, WN, WM, NA, MB, SK, ST>;
    if (lds > kPlainLds) allow_dynamic_lds(kernel, lds, "hipFuncSetAttribute(int8 linear)", __LINE__);
    launch(kernel, dim3(static_cast<unsigned>((tiles * a.splits + 7) / 8 * 8)), dim3(256), lds, st, a);
    if constexpr (KIND == kInt8SplitTile) {
        static_assert(join_lds <= kPlainLds);
        if (a.splits > 1)
            launch(terna_int8_join_kernel<Out, WN, WM, NA, MB, SK, ST>, dim3(static_cast<unsigned>((tiles + 7) / 8 * 8)), dim3(256), join_lds, st, a);
    }
}
template <typename Out>
void launch_int8_linear(const Int8Linear& a, const Int8Plan& plan, hipStream_t st)
{
    switch (plan.tile) {                       // (the order of kInt8Tiles)
    case 0: return launch_int8<Out, 0, 4, 1, 1, 1, 2, 4>(a, plan.tiles, st);
    case 1: return launch_int8<Out, 1, 2, 2, 1, 1, 2, 5>(a, plan.tiles, st);
    case 2: return launch_int8<Out, 2, 4, 1, 1, 2, 1, 6>(a, plan.tiles, st);
    case 3: return launch_int8<Out, 3, 4, 1, 2, 2, 1, 4>(a, plan.tiles, st);
    case 4: return launch_int8<Out, 4, 2, 2, 2, 2, 1, 5>(a, plan.tiles, st);
    case 5: return launch_int8<Out, 5, 2, 2, 2, 3, 1, 4>(a, plan.tiles, st);
    default: return launch_int8<Out, 6, 2, 2, 2, 4, 1, 3>(a, plan.tiles, st);
    }
}
bool int8_linear_ok(int M, int N, int K)
{
    return int8_rows_ok(M, K) && int8_rows_ok(N, K) && launch_fits(int8_plan(M, N, K, true).tiles * kInt8MaxSplits + 8, 256);
}

}  // namespace

extern "C" {

long long ternaspmm_int8_bytes(int R, int K) { return int8_rows_ok(R, K) ? int8_bands(R) * int8_k_blocks(K) * 1024 : -1; }

int ternaspmm_int8_quantise(const void* x, long long row, int fp32, void* packed, float* scale, int R, int K, terna_stream stream)
{
    if (!int8_rows_ok(R, K) || !x || !packed || !scale || !aligned16(packed) || (reinterpret_cast<uintptr_t>(x) & (fp32 ? 3 : 1)) || row < 0 || !launch_fits((R + 31ll) / 32 * 8, kInt8Threads))
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
    const long long waves = int8_bands(R) * ((int8_k_blocks(K) + kInt8PackBlocks - 1) / kInt8PackBlocks), groups = (waves + kInt8Threads / 64 - 1) / (kInt8Threads / 64);
    if (!int8_rows_ok(R, K) || !x || !packed || !aligned16(packed) || row < 0 || !launch_fits(groups, kInt8Threads)) return -1;
    launch(terna_int8_pack_kernel, dim3(static_cast<unsigned>(groups)), dim3(kInt8Threads), 0, static_cast<hipStream_t>(stream), static_cast<const uint8_t*>(x), row,
           static_cast<uint8_t*>(packed), R, K, aligned16(x) && (row & 15) == 0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_int8_pack", e, __LINE__);
    return 0;
}

long long ternaspmm_int8_linear_workspace_bytes(int M, int N, int K)
{
    if (!int8_linear_ok(M, N, K)) return -1;
    const Int8Plan plan = int8_plan(M, N, K, true);
    return plan.splits == 1 ? 0 : 4ll * plan.tiles * plan.splits * kInt8Tiles[plan.tile].features * kInt8Tiles[plan.tile].rows;
}

int ternaspmm_int8_linear(const void* x, const float* x_scale, const void* w, const float* w_scale, void* out, int fp32, void* workspace, int M, int N, int K, terna_stream stream)
{
    if (!int8_linear_ok(M, N, K) || !x || !x_scale || !w || !w_scale || !out || !aligned16(x) || !aligned16(w) || !aligned16(out) || !aligned16(workspace)) return -1;
    const Int8Plan plan = int8_plan(M, N, K, workspace != nullptr);
    const Int8TileTime& tile = kInt8Tiles[plan.tile];
    Int8Linear a{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), x_scale, w_scale, out, static_cast<int32_t*>(workspace), M, N, K,
                 (M + tile.rows - 1) / tile.rows, (N + tile.features - 1) / tile.features, plan.splits};
    if (fp32) launch_int8_linear<float>(a, plan, static_cast<hipStream_t>(stream));
    else launch_int8_linear<uint16_t>(a, plan, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_int8_linear", e, __LINE__);
    return 0;
}

}  // extern "C"
