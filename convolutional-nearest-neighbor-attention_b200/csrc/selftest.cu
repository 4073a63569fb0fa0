// convnn_b200_selftest_wait_timeout: lets a test watch the bounded mbarrier wait of the
// tensor-core kernels give up, without putting any copy, MMA or second CTA at risk.  The
// kernel is one CTA; thread 0 waits on a barrier that expects one arrival which never comes.
// convnn_b200_selftest_pair_drain: the way out of a CTA pair whose producers stopped at different places of their ring
// (sm100::drain_pair_ring), with copies of a few KB and no MMA.
#include "common.cuh"
#include "sm100.cuh"

namespace convnn {
int check_device_is_sm100();
namespace {

__global__ void wait_timeout_kernel(int* status, unsigned long long* waited_ns, unsigned long long budget_ns) {
    __shared__ uint64_t bar;
    __shared__ int abort_flag;
    if (threadIdx.x == 0) {
        sm100::mbar_init(&bar, 1);
        abort_flag = 0;
        sm100::fence_barrier_init();
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned long long t0 = sm100::global_timer_ns();
        const bool ok = sm100::mbar_wait(&bar, 0, &abort_flag, budget_ns);
        *waited_ns = sm100::global_timer_ns() - t0;
        *status = ok ? 0 : 41;
    }
}

// Two CTAs fill the stages of a ring with rows of src, as often as each is told (at most twice round); the first time round is seen to
// land, what both did of it, then nothing is waited for until the drain.  dst: each CTA's stages as they are after it.
constexpr int kDrainStages = 4, kDrainRows = 16, kDrainBytes = kDrainRows * 128;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(128)
pair_drain_kernel(const __grid_constant__ CUtensorMap tm, int fills_even, int fills_odd, uint4* dst, int* status) {
    using namespace sm100;
    __shared__ __align__(1024) uint8_t ring[kDrainStages][kDrainBytes];
    __shared__ uint64_t full[kDrainStages];
    const uint32_t rank = cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kDrainStages; ++s) mbar_init(&full[s], 1);
        fence_barrier_init();
    }
    for (int i = threadIdx.x; i < (int)sizeof(ring) / 16; i += blockDim.x) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    __syncthreads();
    cluster_sync_all();
    const uint32_t full0 = smem_u32(full), lead0 = map_to_cta(full0, 0);
    const int fills = rank == 0 ? fills_even : fills_odd;
    int failed = 0;
    for (int round = 0; round < 2; ++round) {
        if (threadIdx.x == 0) {
            for (int f = round * kDrainStages; f < fills && f < (round + 1) * kDrainStages; ++f) {
                const int s = f % kDrainStages;
                if (rank == 0) mbar_expect_tx_a(full0 + 8 * s, 2 * kDrainBytes);
                tma_load_2d_pair(smem_u32(ring[s]), &tm, lead0 + 8 * s, 0, (f * 2 + (int)rank) * kDrainRows);
            }
            if (rank == 0 && round == 0) {
                int never = 0;
                for (int s = 0; s < kDrainStages && s < fills_even && s < fills_odd; ++s)
                    if (!mbar_wait_a(full0 + 8 * s, 0, &never)) failed = 1;
            }
        }
        __syncwarp();
        cluster_sync_all();
    }
    if (threadIdx.x == 0 && rank == 0) {
        if (!drain_pair_ring(full0, kDrainStages, kDrainBytes, (uint32_t)fills_even, (uint32_t)fills_odd)) failed = 1;
        *status = failed;
    }
    __syncwarp();
    cluster_sync_all();
    for (int i = threadIdx.x; i < (int)sizeof(ring) / 16; i += blockDim.x)
        dst[rank * (sizeof(ring) / 16) + i] = reinterpret_cast<const uint4*>(ring)[i];
}

}  // namespace
}  // namespace convnn

extern "C" int convnn_b200_selftest_wait_timeout(uint32_t budget_us, int* status_dev, uint64_t* waited_ns_dev,
                                                 void* stream) {
    using namespace convnn;
    if (!status_dev || !waited_ns_dev)
        return set_error(CONVNN_E_NULL, "convnn_b200_selftest_wait_timeout: NULL output pointer");
    if (budget_us < 1 || budget_us > 100000)
        return set_error(CONVNN_E_INVALID, "convnn_b200_selftest_wait_timeout: budget_us must be in 1 .. 100000");
    wait_timeout_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(
        status_dev, reinterpret_cast<unsigned long long*>(waited_ns_dev), (unsigned long long)budget_us * 1000ull);
    CONVNN_CHECK_LAUNCH("selftest_wait_timeout");
    return CONVNN_OK;
}

extern "C" int convnn_b200_selftest_pair_drain(int32_t fills_even, int32_t fills_odd, const void* src_dev, void* dst_dev, int* status_dev,
                                               void* stream) {
    using namespace convnn;
    if (!src_dev || !dst_dev || !status_dev) return set_error(CONVNN_E_NULL, "convnn_b200_selftest_pair_drain: a pointer is NULL");
    if (fills_even < 0 || fills_odd < 0 || fills_even > 2 * kDrainStages || fills_odd > 2 * kDrainStages ||
        (fills_even > kDrainStages && fills_odd < fills_even - kDrainStages) ||
        (fills_odd > kDrainStages && fills_even < fills_odd - kDrainStages))
        return set_error(CONVNN_E_INVALID, "convnn_b200_selftest_pair_drain: fills must be in 0 .. 8 and at most 4 apart, got %d and %d",
                         fills_even, fills_odd);
    if (!aligned16(src_dev) || !aligned16(dst_dev) || (reinterpret_cast<uintptr_t>(status_dev) & 3u))
        return set_error(CONVNN_E_ALIGN, "convnn_b200_selftest_pair_drain: src and dst must be 16-byte aligned");
    if (const int rc = check_device_is_sm100()) return rc;
    CUtensorMap tm;
    const uint64_t dims[2] = {128, 2 * 2 * kDrainStages * kDrainRows}, strides[1] = {128};
    const uint32_t box[2] = {128, kDrainRows};
    if (!encode_tensor_map_u8(&tm, src_dev, 2, dims, strides, box, 0)) return CONVNN_E_CUDA;
    pair_drain_kernel<<<2, 128, 0, static_cast<cudaStream_t>(stream)>>>(tm, fills_even, fills_odd, static_cast<uint4*>(dst_dev), status_dev);
    CONVNN_CHECK_LAUNCH("selftest_pair_drain");
    return CONVNN_OK;
}
