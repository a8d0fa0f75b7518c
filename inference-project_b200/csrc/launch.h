// Launching the stand-alone kernels of the paged-cache operators: every one waits (griddepcontrol.wait) before
// it touches memory, so it may be launched while the kernel before it on the stream drains, and lets the
// next one start only behind that wait.  Memory is visible to the grid that waits and no other: a kernel that
// counted on the wait of the one before it would read without a promise, though that one had completed.
#pragma once

#include <mutex>
#include <set>
#include <utility>

#include "runtime.h"

namespace inf {

template <typename... KArgs, typename... Args>
Error_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args)
{
	cudaLaunchConfig_t lc = {};
	lc.gridDim = grid;
	lc.blockDim = block;
	lc.dynamicSmemBytes = smem;
	lc.stream = stream;
	cudaLaunchAttribute attr[1];
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[0].val.programmaticStreamSerializationAllowed = 1;
	lc.attrs = attr;
	lc.numAttrs = 1;
	INF_CUDA_TRY(cudaLaunchKernelEx(&lc, kern, std::forward<Args>(args)...));
	return Success;
}

// Raises a kernel's dynamic shared-memory ceiling once per device (`bytes`: the most any launch of it
// asks for).
template <typename K>
Error_t allow_smem(K kern, size_t bytes)
{
	static std::mutex m;
	static std::set<std::pair<const void*, int>> done;
	int dev = 0;
	INF_CUDA_TRY(cudaGetDevice(&dev));
	const std::pair<const void*, int> key(reinterpret_cast<const void*>(kern), dev);
	std::lock_guard<std::mutex> lk(m);
	if (done.count(key)) return Success;
	INF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
	done.insert(key);
	return Success;
}

// Multiprocessors of the current device.
Error_t sm_count(int* out);

// The checks every operator of a caller's paged cache shares: the shapes of *kv (and of its block
// table, where it is used) and `layer`; then its device pointers.
Error_t check_paged_kv(const char* who, const InfPagedKv* kv, u32 layer, bool table);
Error_t check_paged_kv_pointers(const char* who, const InfPagedKv* kv, bool table, bool refs);
// A device pointer argument of such an operator, aligned to `align` bytes.
Error_t check_dev_arg(const char* who, const char* name, const void* p, u64 align);
Error_t check_status_arg(const char* who, const i32* status);

} // namespace inf
