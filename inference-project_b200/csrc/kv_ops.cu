// Entry points of the paged-cache operators besides attention: the norm + rotation + cache write of
// new tokens, and copying, freeing, forking and compacting pages.  They enqueue work on the caller's
// stream and return; nothing is allocated or synchronised.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "k_kv_pages.cuh"
#include "k_qk_norm_rope.cuh"
#include "launch.h"

namespace inf {

Error_t sm_count(int* out)
{
	int dev = 0;
	INF_CUDA_TRY(cudaGetDevice(&dev));
	INF_CUDA_TRY(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
	return Success;
}

Error_t check_dev_arg(const char* who, const char* name, const void* p, u64 align)
{
	if ((uintptr_t)p & (align - 1)) return fail(ErrorInvalidValue, "%s: %s not %llu-byte aligned", who, name, (unsigned long long)align);
	if (!is_local_device_ptr(p)) return fail(ErrorInvalidDevPtr, "%s: %s is not memory of the current device", who, name);
	return Success;
}

Error_t check_status_arg(const char* who, const i32* status)
{
	return status ? check_dev_arg(who, "status", status, 4) : Success;
}

Error_t check_paged_kv(const char* who, const InfPagedKv* kv, u32 layer, bool table)
{
	if (!kv) return fail(ErrorInvalidValue, "%s: no cache", who);
	const u64 es = kv->dtype == InfBF16 ? 2 : 4;
	if ((kv->dtype != InfBF16 && kv->dtype != InfF32) || kv->n_pages == 0 || kv->n_pages > 0x7FFFFFFFu || kv->n_layers == 0 ||
	    kv->n_kv_heads == 0 || kv->n_kv_heads > 65535 || kv->head_dim == 0 || kv->head_dim > 65536 || kv->kv_block == 0 ||
	    kv->kv_block > 65536)
		return fail(ErrorInvalidValue, "%s: bad cache shape", who);
	if ((kv->head_dim * es) % 16) return fail(ErrorUnsupported, "%s: head_dim %u: rows are not a multiple of 16 bytes", who, kv->head_dim);
	const u64 page_bytes = (u64)kv->n_kv_heads * kv->kv_block * kv->head_dim * es;
	if (page_bytes > 0x7FFFFFFFull) return fail(ErrorUnsupported, "%s: pages of 2 GB and more", who);
	if (layer >= kv->n_layers) return fail(ErrorInvalidValue, "%s: layer %u of %u", who, layer, kv->n_layers);
	if (kv->n_layers > 1 && (kv->layer_stride % 16 || kv->layer_stride < page_bytes * kv->n_pages))
		return fail(ErrorInvalidValue, "%s: layer_stride", who);
	if (table && (kv->n_slots == 0 || kv->n_slots > 0x7FFFFFFFu || kv->pages_per_seq == 0 ||
	              (u64)kv->pages_per_seq * kv->kv_block > (1ull << 30)))
		return fail(ErrorInvalidValue, "%s: bad block table shape", who);
	return Success;
}

Error_t check_paged_kv_pointers(const char* who, const InfPagedKv* kv, bool table, bool refs)
{
	INF_TRY(check_dev_arg(who, "kpool", kv->kpool, 16));
	INF_TRY(check_dev_arg(who, "vpool", kv->vpool, 16));
	if (table) INF_TRY(check_dev_arg(who, "block_table", kv->block_table, 4));
	if (refs) INF_TRY(check_dev_arg(who, "page_refs", kv->page_refs, 4));
	return Success;
}

} // namespace inf

using namespace inf;

namespace {

PagePools page_pools(const InfPagedKv* kv)
{
	PagePools P;
	P.k = (uint8_t*)kv->kpool;
	P.v = (uint8_t*)kv->vpool;
	P.layer_stride = kv->n_layers > 1 ? kv->layer_stride : 0;
	P.n_layers = kv->n_layers;
	P.row_bytes = kv->head_dim * (kv->dtype == InfBF16 ? 2 : 4);
	P.head_bytes = P.row_bytes * kv->kv_block;
	P.page_bytes = P.head_bytes * kv->n_kv_heads;
	P.n_pages = (int)kv->n_pages;
	return P;
}

// The kernels count a page's pieces (slices of K and V, or heads, over all layers) in 32 bits.
Error_t check_page_pieces(const char* who, const InfPagedKv* kv)
{
	const PagePools P = page_pools(kv);
	const u64 slices = ((u64)P.page_bytes + kPgSlice - 1) / kPgSlice;
	if (2 * (u64)kv->n_layers * std::max<u64>(slices, kv->n_kv_heads) > 0x7FFFFFFFull)
		return fail(ErrorUnsupported, "%s: %u layers of %u bytes a page", who, kv->n_layers, P.page_bytes);
	return Success;
}

// CTAs of a copy of `bytes`: a warp per slice up to eight CTAs on every SM.
unsigned copy_ctas(u64 bytes, int sms)
{
	const u64 ctas = (bytes + (u64)kPgSlice * (kPgThreads / kWarp) - 1) / ((u64)kPgSlice * (kPgThreads / kWarp));
	return (unsigned)std::max<u64>(1, std::min<u64>(ctas, (u64)sms * 8));
}

u64 up16(u64 n) { return (n + 15) & ~15ull; }

template <typename T>
Error_t launch_qk_norm_rope(QkNormRopeArgs& a, int sms, cudaStream_t st)
{
	const int half_units = a.hd / Store<T>::kVec / 2;
	const int vp = half_units > kWarp ? 2 : 1; // head_dim <= 512: at most 64 unit pairs
	a.lanes = 1;
	while (a.lanes * vp < half_units) a.lanes <<= 1;
	const int heads = a.H + 2 * a.KV;
	// A warp takes all heads of its token where there are tokens enough to fill the SMs (24 warps each); with
	// fewer, as few heads as its groups hold at a time, so that a decode step's heads run side by side.
	const int groups = kWarp / a.lanes;
	a.chunk = heads;
	while (a.chunk > groups && (u64)a.n_tokens * ((heads + a.chunk - 1) / a.chunk) < (u64)sms * 24) a.chunk = std::max(groups, (a.chunk + 1) / 2);
	a.chunks = (heads + a.chunk - 1) / a.chunk;
	const u64 ctas = ((u64)a.n_tokens * a.chunks + kQnThreads / kWarp - 1) / (kQnThreads / kWarp);
	if (ctas > 0x7FFFFFFFull) return fail(ErrorUnsupported, "inf_qk_norm_rope: %u tokens of %d heads", a.n_tokens, heads);
	return launch_pdl(vp == 2 ? k_qk_norm_rope_rows<T, 2> : k_qk_norm_rope_rows<T, 1>, dim3((unsigned)ctas), dim3(kQnThreads), 0, st, a);
}

} // namespace

extern "C" {

Error_t inf_check_status(i32* d_status, void* stream)
{
	INF_TRY(check_dev_arg("inf_check_status", "status", d_status, 4));
	// a wait would invalidate the capture
	cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
	INF_CUDA_TRY(cudaStreamIsCapturing((cudaStream_t)stream, &capture));
	if (capture != cudaStreamCaptureStatusNone) return fail(ErrorInvalidValue, "inf_check_status: the stream is capturing");
	i32 v = 0;
	INF_CUDA_TRY(cudaMemcpyAsync(&v, d_status, sizeof v, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
	INF_CUDA_TRY(cudaMemsetAsync(d_status, 0, sizeof v, (cudaStream_t)stream));
	INF_CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
	return map_dev_err(v);
}

Error_t inf_qk_norm_rope(const InfPagedKv* kv, const InfQkNormRope* args, void* stream)
{
	const char* who = "inf_qk_norm_rope";
	if (!args) return fail(ErrorInvalidValue, "%s: no arguments", who);
	const InfQkNormRope& A = *args;
	INF_TRY(check_paged_kv(who, kv, A.layer, true));
	const u64 es = kv->dtype == InfBF16 ? 2 : 4, hd = kv->head_dim;
	if (A.n_heads == 0 || A.n_heads > 65535 || A.n_pos == 0 || A.n_pos > 0x7FFFFFFFu || A.n_tokens > 0x7FFFFFFFu)
		return fail(ErrorInvalidValue, "%s: bad shape", who);
	if ((hd * es) % 32 || hd > 512) return fail(ErrorUnsupported, "%s: head_dim %u", who, kv->head_dim);
	const u64 qkv_row = (u64)(A.n_heads + 2 * kv->n_kv_heads) * hd, q_row = (u64)A.n_heads * hd;
	const u64 qs = A.qkv_stride ? A.qkv_stride : qkv_row, os = A.q_out_stride ? A.q_out_stride : q_row;
	if (qs < qkv_row || os < q_row || qs > (1ull << 40) || os > (1ull << 40) || (qs * es) % 16 || (os * es) % 16)
		return fail(ErrorInvalidValue, "%s: row strides", who);
	if (!(A.eps >= 0.0f) || !std::isfinite(A.eps) || !std::isfinite(A.gain_offset))
		return fail(ErrorInvalidValue, "%s: eps %g, gain_offset %g", who, A.eps, A.gain_offset);
	if (A.n_tokens == 0) return Success;
	if (A.qkv == A.q_out && qs != os) return fail(ErrorInvalidValue, "%s: in place needs equal strides", who);
	INF_TRY(check_paged_kv_pointers(who, kv, true, false));
	INF_TRY(check_dev_arg(who, "qkv", A.qkv, 16));
	INF_TRY(check_dev_arg(who, "q_out", A.q_out, 16));
	if (A.q_gain) INF_TRY(check_dev_arg(who, "q_gain", A.q_gain, 16));
	if (A.k_gain) INF_TRY(check_dev_arg(who, "k_gain", A.k_gain, 16));
	INF_TRY(check_dev_arg(who, "rope_cos", A.rope_cos, 16));
	INF_TRY(check_dev_arg(who, "rope_sin", A.rope_sin, 16));
	INF_TRY(check_dev_arg(who, "tok_slot", A.tok_slot, 4));
	INF_TRY(check_dev_arg(who, "tok_pos", A.tok_pos, 4));
	INF_TRY(check_status_arg(who, A.status));
	int sms = 0;
	INF_TRY(sm_count(&sms));
	QkNormRopeArgs a;
	memset(&a, 0, sizeof a);
	a.qkv = (const uint8_t*)A.qkv;
	a.q_out = (uint8_t*)A.q_out;
	a.qkv_stride = qs * es;
	a.q_out_stride = os * es;
	a.q_gain = A.q_gain;
	a.k_gain = A.k_gain;
	a.rope_cos = A.rope_cos;
	a.rope_sin = A.rope_sin;
	a.tok_slot = A.tok_slot;
	a.tok_pos = A.tok_pos;
	a.status = A.status;
	a.eps = A.eps;
	a.gain_offset = A.gain_offset;
	a.inv_hd = (float)(1.0 / (double)hd);
	a.n_pos = (int)A.n_pos;
	a.n_tokens = A.n_tokens;
	a.H = (int)A.n_heads;
	a.KV = (int)kv->n_kv_heads;
	a.hd = (int)hd;
	a.blk = (int)kv->kv_block;
	const u64 off = kv->n_layers > 1 ? (u64)A.layer * kv->layer_stride : 0;
	a.kpool = (uint8_t*)kv->kpool + off;
	a.vpool = (uint8_t*)kv->vpool + off;
	a.table = kv->block_table;
	a.n_slots = (int)kv->n_slots;
	a.pages_per_seq = (int)kv->pages_per_seq;
	a.n_pages = (int)kv->n_pages;
	return kv->dtype == InfBF16 ? launch_qk_norm_rope<bf16>(a, sms, (cudaStream_t)stream)
	                            : launch_qk_norm_rope<float>(a, sms, (cudaStream_t)stream);
}

Error_t inf_kv_copy_pages(const InfPagedKv* kv, const i32* d_src, const i32* d_dst, u32 n, i32* d_status, void* stream)
{
	const char* who = "inf_kv_copy_pages";
	INF_TRY(check_paged_kv(who, kv, 0, false));
	INF_TRY(check_page_pieces(who, kv));
	if (n > kv->n_pages) return fail(ErrorInvalidValue, "%s: %u pairs in %u pages", who, n, kv->n_pages);
	if (n == 0) return Success;
	INF_TRY(check_paged_kv_pointers(who, kv, false, false));
	INF_TRY(check_dev_arg(who, "src", d_src, 4));
	INF_TRY(check_dev_arg(who, "dst", d_dst, 4));
	INF_TRY(check_status_arg(who, d_status));
	int sms = 0;
	INF_TRY(sm_count(&sms));
	PageCopyArgs a = {page_pools(kv), d_src, d_dst, n, d_status};
	return launch_pdl(k_kv_copy_pages, dim3(copy_ctas((u64)n * 2 * kv->n_layers * a.P.page_bytes, sms)), dim3(kPgThreads), 0,
	                  (cudaStream_t)stream, a);
}

Error_t inf_kv_free(const InfPagedKv* kv, const i32* d_slot, const i32* d_first, const i32* d_last, u32 n, i32* d_status,
                    void* stream)
{
	const char* who = "inf_kv_free";
	INF_TRY(check_paged_kv(who, kv, 0, true));
	if (n > 0x7FFFFFFFu) return fail(ErrorInvalidValue, "%s: %u ranges", who, n);
	if (n == 0) return Success;
	INF_TRY(check_paged_kv_pointers(who, kv, true, true));
	INF_TRY(check_dev_arg(who, "slot", d_slot, 4));
	if (d_first) INF_TRY(check_dev_arg(who, "first", d_first, 4));
	if (d_last) INF_TRY(check_dev_arg(who, "last", d_last, 4));
	INF_TRY(check_status_arg(who, d_status));
	PageFreeArgs a = {kv->block_table, kv->page_refs, (int)kv->n_slots, (int)kv->pages_per_seq, (int)kv->n_pages,
	                  d_slot, d_first, d_last, d_status};
	const unsigned gx = std::min<unsigned>((kv->pages_per_seq + kPgThreads - 1) / kPgThreads, 64u);
	return launch_pdl(k_kv_free, dim3(gx, std::min<unsigned>(n, 65535u)), dim3(kPgThreads), 0, (cudaStream_t)stream, a, (uint32_t)n);
}

u64 inf_kv_pages_scratch_bytes(const InfPagedKv* kv)
{
	if (!kv) return 0;
	const u64 fork = up16((u64)kv->n_slots * sizeof(ForkJob)) + (u64)kv->n_slots * 4;
	const u64 compact = 16 + 2 * up16((u64)kv->n_pages * 4);
	return up16(std::max(fork, compact));
}

Error_t inf_kv_fork(const InfPagedKv* kv, const i32* d_src, const i32* d_dst, const i32* d_len, u32 n, void* d_scratch,
                    u64 scratch_bytes, i32* d_status, void* stream)
{
	const char* who = "inf_kv_fork";
	INF_TRY(check_paged_kv(who, kv, 0, true));
	INF_TRY(check_page_pieces(who, kv));
	if (n > kv->n_slots) return fail(ErrorInvalidValue, "%s: %u forks into %u slots", who, n, kv->n_slots);
	if (n == 0) return Success;
	if (scratch_bytes < inf_kv_pages_scratch_bytes(kv)) return fail(ErrorInvalidValue, "%s: scratch too small", who);
	INF_TRY(check_paged_kv_pointers(who, kv, true, true));
	INF_TRY(check_dev_arg(who, "src", d_src, 4));
	INF_TRY(check_dev_arg(who, "dst", d_dst, 4));
	INF_TRY(check_dev_arg(who, "len", d_len, 4));
	INF_TRY(check_dev_arg(who, "scratch", d_scratch, 16));
	INF_TRY(check_status_arg(who, d_status));
	int sms = 0;
	INF_TRY(sm_count(&sms));
	ForkArgs a;
	memset(&a, 0, sizeof a);
	a.P = page_pools(kv);
	a.table = kv->block_table;
	a.refs = kv->page_refs;
	a.n_slots = (int)kv->n_slots;
	a.pages_per_seq = (int)kv->pages_per_seq;
	a.kv_block = (int)kv->kv_block;
	a.src = d_src;
	a.dst = d_dst;
	a.len = d_len;
	a.n = n;
	a.jobs = (ForkJob*)d_scratch;
	a.fresh = (int*)((uint8_t*)d_scratch + up16((u64)kv->n_slots * sizeof(ForkJob)));
	a.status = d_status;
	const cudaStream_t st = (cudaStream_t)stream;
	INF_TRY(launch_pdl(k_kv_fork_plan, dim3(1), dim3(kPlanThreads), 0, st, a));
	const u64 segs = (u64)n * 2 * kv->n_layers * kv->n_kv_heads;
	const unsigned ctas = (unsigned)std::min<u64>((segs + kPgThreads / kWarp - 1) / (kPgThreads / kWarp), (u64)sms * 8);
	return launch_pdl(k_kv_fork, dim3(n + ctas), dim3(kPgThreads), 0, st, a);
}

Error_t inf_kv_compact(const InfPagedKv* kv, i32* d_map, i32* d_n_live, void* d_scratch, u64 scratch_bytes, i32* d_status,
                       void* stream)
{
	const char* who = "inf_kv_compact";
	INF_TRY(check_paged_kv(who, kv, 0, true));
	INF_TRY(check_page_pieces(who, kv));
	if (kv->n_pages > kCompactMaxPages) return fail(ErrorUnsupported, "%s: %u pages, above %u", who, kv->n_pages, kCompactMaxPages);
	if (scratch_bytes < inf_kv_pages_scratch_bytes(kv)) return fail(ErrorInvalidValue, "%s: scratch too small", who);
	INF_TRY(check_paged_kv_pointers(who, kv, true, true));
	INF_TRY(check_dev_arg(who, "map", d_map, 4));
	INF_TRY(check_dev_arg(who, "n_live", d_n_live, 4));
	INF_TRY(check_dev_arg(who, "scratch", d_scratch, 16));
	INF_TRY(check_status_arg(who, d_status));
	int sms = 0;
	INF_TRY(sm_count(&sms));
	CompactArgs a;
	memset(&a, 0, sizeof a);
	a.P = page_pools(kv);
	a.table = kv->block_table;
	a.refs = kv->page_refs;
	a.n_slots = (int)kv->n_slots;
	a.pages_per_seq = (int)kv->pages_per_seq;
	a.map = d_map;
	a.n_live = d_n_live;
	a.n_moves = (int*)d_scratch;
	a.from = (int*)((uint8_t*)d_scratch + 16);
	a.to = (int*)((uint8_t*)d_scratch + 16 + up16((u64)kv->n_pages * 4));
	a.status = d_status;
	const cudaStream_t st = (cudaStream_t)stream;
	const size_t smem = (size_t)((kv->n_pages + 31) / 32) * 8;
	INF_TRY(allow_smem(k_kv_compact_plan, (size_t)kCompactMaxPages / 32 * 8));
	INF_TRY(launch_pdl(k_kv_compact_plan, dim3(1), dim3(kPlanThreads), smem, st, a));
	return launch_pdl(k_kv_compact, dim3(copy_ctas((u64)kv->n_pages * 2 * kv->n_layers * a.P.page_bytes, sms)), dim3(kPgThreads), 0,
	                  st, a);
}

} // extern "C"
