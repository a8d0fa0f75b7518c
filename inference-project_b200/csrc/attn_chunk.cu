// inf_attn_chunk: attention of a ragged batch of new tokens over the paged cache.  Chooses the kernels
// and their number of workers from what the host knows (types, head layout, row counts at most), lays
// out the scratch, and enqueues them.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "k_attn_chunk.cuh"
#include "k_attn_chunk_rows.cuh"
#include "k_attn_chunk_tc.cuh"
#include "launch.h"

using namespace inf;

namespace {

u64 up256(u64 n) { return (n + 255) & ~255ull; }

// One kernel's share of a call: the sequences with rows_min < rows <= rows_max rows per KV head.
struct ChunkPass {
	enum Kind { F32, Rows, TC } kind;
	int rows_min, rows_max;
	int workers, min_run, item_cost;
	int R;               // row tile
	size_t smem;
	u64 part_off, jobs_off;
};

struct ChunkPlan {
	ChunkPass pass[2];
	int n_pass;
	u64 scratch;
};

// Items times their cost at most.
u64 units_max(const InfPagedKv* kv, u32 n_heads, u32 n_tokens, u32 n_seqs, u32 R, u32 KT, u32 item_cost)
{
	const u64 G = n_heads / kv->n_kv_heads;
	const u64 tiles = (u64)n_tokens * G / R + std::min(n_seqs, n_tokens);
	return tiles * kv->n_kv_heads * (((u64)kv->pages_per_seq * kv->kv_block + KT - 1) / KT + 1 + item_cost);
}

Error_t chunk_plan(const InfPagedKv* kv, u32 n_heads, u32 n_tokens, u32 n_seqs, ChunkPlan* P)
{
	const char* who = "inf_attn_chunk";
	if (n_heads == 0 || n_heads > 65535 || n_heads % kv->n_kv_heads || n_seqs > (u32)kAcMaxSeqs ||
	    (u64)n_tokens * (n_heads / kv->n_kv_heads) > (1u << 30))
		return fail(ErrorInvalidValue, "%s: %u heads on %u KV heads, %u sequences, %u tokens", who, n_heads, kv->n_kv_heads, n_seqs,
		            n_tokens);
	const u64 es = kv->dtype == InfBF16 ? 2 : 4;
	if (kv->head_dim > 512 || (kv->head_dim * es) % 16)
		return fail(ErrorUnsupported, "%s: head_dim %u", who, kv->head_dim);
	int sms = 148; // the scratch size is also asked for without a device
	(void)sm_count(&sms);
	P->n_pass = 0;
	P->scratch = 0;
	// The scratch is laid out for `most` workers, which do not depend on n_seqs: a call of fewer sequences, whose
	// smaller prefix lets more workers onto an SM, fits where a call of more did.
	auto add = [&](ChunkPass p, u64 units, int most) -> Error_t {
		if (units > 0x7FFFFFFFull) return fail(ErrorUnsupported, "%s: %u tokens of %u positions at most", who, n_tokens, kv->pages_per_seq * kv->kv_block);
		const u64 runs = std::max<u64>(1, (units + p.min_run - 1) / p.min_run), room = std::min<u64>(most, runs);
		p.workers = (int)std::min<u64>(p.workers, runs);
		p.part_off = P->scratch;
		P->scratch += up256(2 * room * ac_part_floats(p.R, (int)kv->head_dim) * sizeof(float));
		p.jobs_off = P->scratch;
		P->scratch += up256(room * kAcJobInts * sizeof(int));
		P->pass[P->n_pass++] = p;
		return Success;
	};
	const u32 blk = kv->kv_block, G = n_heads / kv->n_kv_heads;
	if (kv->dtype == InfBF16 && G <= kCtRows && (kv->head_dim == 64 || kv->head_dim == 128) &&
	    (blk == 16 || blk == 32 || blk == 64 || blk == 128)) {
		// Sequences of at most 16 rows per KV head go to the streaming kernel (HBM-bound, a warp per worker), longer
		// ones to the tensor-core kernel, which reads K and V as fast but computes 128 rows whatever is there.
		// Where sequences of max_new rows nearly fill the tokens no short one is left, and the tensor-core
		// kernel takes all: the other launch would cost 3 us for nothing.
		if (G <= (u32)kCrRows) {
			ChunkPass r = {};
			r.kind = ChunkPass::Rows;
			r.rows_max = kCrRows;
			r.R = kCrRows;
			r.min_run = 4;
			r.smem = attn_chunk_rows_smem((int)kv->head_dim, (int)n_seqs);
			r.workers = sms * kCrWarps;
			INF_TRY(add(r, (u64)std::min(n_seqs, n_tokens) * kv->n_kv_heads * (((u64)kv->pages_per_seq * blk + kCrKT - 1) / kCrKT + 1), r.workers));
		}
		ChunkPass t = {};
		t.kind = ChunkPass::TC;
		t.rows_min = G <= (u32)kCrRows ? kCrRows : 0;
		t.rows_max = 0x7FFFFFFF;
		t.R = (int)(2 * (kCtRows / G) * G); // whole tokens in each half
		t.item_cost = kCtItemCost;
		t.min_run = 2 + kCtItemCost;
		t.smem = ct_layout((int)kv->head_dim, (int)n_seqs).total;
		t.workers = sms;
		return add(t, units_max(kv, n_heads, n_tokens, n_seqs, (u32)t.R, kCtKT, kCtItemCost), t.workers);
	}
	ChunkPass f = {};
	f.kind = ChunkPass::F32;
	f.rows_max = 0x7FFFFFFF;
	f.R = kAfR;
	f.min_run = 2;
	f.smem = attn_chunk_f32_smem((int)kv->head_dim, (int)n_seqs);
	auto ctas = [&](size_t smem) { return sms * (int)std::max<u64>(1, std::min<u64>(8, (200u << 10) / smem)); };
	f.workers = ctas(f.smem);
	return add(f, units_max(kv, n_heads, n_tokens, n_seqs, kAfR, kAfKT, 0), ctas(attn_chunk_f32_smem((int)kv->head_dim, 0)));
}

template <typename T>
Error_t launch_f32(const AttnChunkArgs& a, const ChunkPass& p, cudaStream_t st)
{
	void (*k)(const AttnChunkArgs) = a.hd <= 128 ? k_attn_chunk_f32<T, 1> : a.hd <= 256 ? k_attn_chunk_f32<T, 2> : k_attn_chunk_f32<T, 4>;
	INF_TRY(allow_smem(k, attn_chunk_f32_smem(a.hd <= 128 ? 128 : a.hd <= 256 ? 256 : 512, kAcMaxSeqs)));
	return launch_pdl(k, dim3((unsigned)p.workers), dim3(kAfThreads), p.smem, st, a);
}

template <int HD>
Error_t launch_tc(const AttnChunkArgs& a, const ChunkPass& p, cudaStream_t st)
{
	const u32 blk = (u32)a.blk, box = kCtKT / blk;
	CUtensorMap q, k8, k1, v8, v1;
	INF_TRY(tensor_map_q(&q, a.q, (u32)a.n_tokens, (u32)a.H, HD, a.q_stride, (u32)a.G, (u32)(kCtRows / a.G)));
	INF_TRY(tensor_map_kv_groups(&k8, a.kpool, HD, blk, (u32)a.KV, (u32)a.n_pages, box, blk / 8));
	INF_TRY(tensor_map_kv_groups(&k1, a.kpool, HD, blk, (u32)a.KV, (u32)a.n_pages, 1, blk / 8));
	INF_TRY(tensor_map_kv_groups(&v8, a.vpool, HD, blk, (u32)a.KV, (u32)a.n_pages, box, blk / 8));
	INF_TRY(tensor_map_kv_groups(&v1, a.vpool, HD, blk, (u32)a.KV, (u32)a.n_pages, 1, blk / 8));
	INF_TRY(allow_smem(k_attn_chunk_tc<HD>, 227 * 1024));
	// the kernel's warpgroups trade registers within what it was launched with
	static std::atomic<bool> regs_seen{false};
	if (!regs_seen.load(std::memory_order_relaxed)) {
		cudaFuncAttributes f;
		INF_CUDA_TRY(cudaFuncGetAttributes(&f, k_attn_chunk_tc<HD>));
		if (f.numRegs < kCtRegsLaunch) return fail(ErrorUnsupported, "inf_attn_chunk: built with %d registers a thread", f.numRegs);
		regs_seen.store(true, std::memory_order_relaxed);
	}
	return launch_pdl(k_attn_chunk_tc<HD>, dim3((unsigned)p.workers), dim3(kCtThreads), p.smem, st, q, k8, k1, v8, v1, a);
}

template <int HD>
Error_t launch_rows(const AttnChunkArgs& a, const ChunkPass& p, cudaStream_t st)
{
	CUtensorMap k, v;
	INF_TRY(tensor_map_kv_groups(&k, a.kpool, HD, (u32)a.blk, (u32)a.KV, (u32)a.n_pages, 1, kCrKT / 8));
	INF_TRY(tensor_map_kv_groups(&v, a.vpool, HD, (u32)a.blk, (u32)a.KV, (u32)a.n_pages, 1, kCrKT / 8));
	INF_TRY(allow_smem(k_attn_chunk_rows<HD>, attn_chunk_rows_smem(HD, kAcMaxSeqs)));
	return launch_pdl(k_attn_chunk_rows<HD>, dim3((unsigned)((p.workers + kCrWarps - 1) / kCrWarps)), dim3(kCrThreads), p.smem, st, k, v, a);
}

} // namespace

extern "C" {

u64 inf_attn_chunk_scratch_bytes(const InfPagedKv* kv, u32 n_heads, u32 n_tokens, u32 n_seqs)
{
	ChunkPlan P;
	if (!kv || kv->n_kv_heads == 0 || kv->kv_block == 0 || chunk_plan(kv, n_heads, n_tokens, n_seqs, &P) != Success) return 0;
	return P.scratch;
}

Error_t inf_attn_chunk(const InfPagedKv* kv, const InfAttnChunk* args, void* stream)
{
	const char* who = "inf_attn_chunk";
	if (!args) return fail(ErrorInvalidValue, "%s: no arguments", who);
	const InfAttnChunk& A = *args;
	INF_TRY(check_paged_kv(who, kv, A.layer, true));
	ChunkPlan P;
	INF_TRY(chunk_plan(kv, A.n_heads, A.n_tokens, A.n_seqs, &P));
	const u64 es = kv->dtype == InfBF16 ? 2 : 4, row = (u64)A.n_heads * kv->head_dim;
	const u64 qs = A.q_stride ? A.q_stride : row, os = A.out_stride ? A.out_stride : row;
	if (qs < row || os < row || qs > (1ull << 38) || os > (1ull << 38) || (qs * es) % 16 || (os * es) % 16)
		return fail(ErrorInvalidValue, "%s: row strides", who);
	if (!(A.scale >= 0.0f) || !std::isfinite(A.scale)) return fail(ErrorInvalidValue, "%s: scale %g", who, A.scale);
	if (A.n_seqs == 0 || A.n_tokens == 0) return Success;
	if (A.q == A.out) return fail(ErrorInvalidValue, "%s: out is q", who);
	if (A.scratch_bytes < P.scratch) return fail(ErrorInvalidValue, "%s: scratch needs %llu bytes", who, (unsigned long long)P.scratch);
	INF_TRY(check_paged_kv_pointers(who, kv, true, false));
	INF_TRY(check_dev_arg(who, "q", A.q, 16));
	INF_TRY(check_dev_arg(who, "out", A.out, 16));
	INF_TRY(check_dev_arg(who, "q_start", A.q_start, 4));
	INF_TRY(check_dev_arg(who, "ctx_len", A.ctx_len, 4));
	if (A.seq_slot) INF_TRY(check_dev_arg(who, "seq_slot", A.seq_slot, 4));
	INF_TRY(check_dev_arg(who, "scratch", A.scratch, 16));
	INF_TRY(check_status_arg(who, A.status));
	AttnChunkArgs a;
	memset(&a, 0, sizeof a);
	a.q = A.q;
	a.out = A.out;
	a.q_stride = qs;
	a.out_stride = os;
	const u64 off = kv->n_layers > 1 ? (u64)A.layer * kv->layer_stride : 0;
	a.kpool = (const uint8_t*)kv->kpool + off;
	a.vpool = (const uint8_t*)kv->vpool + off;
	a.table = kv->block_table;
	a.q_start = A.q_start;
	a.ctx_len = A.ctx_len;
	a.seq_slot = A.seq_slot;
	a.n_seqs = (int)A.n_seqs;
	a.n_tokens = (int)A.n_tokens;
	a.max_new = (int)(A.max_new ? std::min(A.max_new, A.n_tokens) : A.n_tokens);
	a.H = (int)A.n_heads;
	a.KV = (int)kv->n_kv_heads;
	a.G = a.H / a.KV;
	a.group = ac_div(a.G);
	a.hd = (int)kv->head_dim;
	a.blk = (int)kv->kv_block;
	a.n_slots = (int)kv->n_slots;
	a.pages_per_seq = (int)kv->pages_per_seq;
	a.n_pages = (int)kv->n_pages;
	// a window that no context outgrows hides nothing
	a.window = A.window >= kv->pages_per_seq * kv->kv_block ? 0 : (int)A.window;
	a.n_sink = (int)std::min(A.n_sink, 1u << 30);
	a.scale = A.scale > 0.0f ? A.scale : (float)(1.0 / std::sqrt((double)kv->head_dim));
	a.status = A.status;
	const cudaStream_t st = (cudaStream_t)stream;
	auto pass_args = [&](const ChunkPass& p) {
		AttnChunkArgs b = a;
		b.rows_min = p.rows_min;
		b.rows_max = p.rows_max;
		b.R = p.R;
		b.workers = p.workers;
		b.min_run = p.min_run;
		b.item_cost = p.item_cost;
		b.part = (float*)((uint8_t*)A.scratch + p.part_off);
		b.jobs = (int*)((uint8_t*)A.scratch + p.jobs_off);
		return b;
	};
	// which of the two bf16 passes can have work
	bool on[2] = {P.n_pass > 0, P.n_pass > 1};
	if (P.n_pass == 2) {
		const u64 slack = (u64)a.n_seqs * (u64)a.max_new - (u64)a.n_tokens; // rows missing to max_new in every sequence
		on[1] = (u64)a.max_new * a.G > (u64)kCrRows;
		on[0] = !on[1] || (u64)a.n_seqs * (u64)a.max_new < (u64)a.n_tokens || (slack + kCrRows / a.G) >= (u64)a.max_new;
		if (!on[0]) P.pass[1].rows_min = 0;
	}
	for (int i = 0; i < P.n_pass; ++i) {
		if (!on[i]) continue;
		const ChunkPass& p = P.pass[i];
		const AttnChunkArgs b = pass_args(p);
		if (p.kind == ChunkPass::Rows) INF_TRY(a.hd == 64 ? launch_rows<64>(b, p, st) : launch_rows<128>(b, p, st));
		else if (p.kind == ChunkPass::TC) INF_TRY(a.hd == 64 ? launch_tc<64>(b, p, st) : launch_tc<128>(b, p, st));
		else INF_TRY(kv->dtype == InfBF16 ? launch_f32<bf16>(b, p, st) : launch_f32<float>(b, p, st));
	}
	for (int i = 0; i < P.n_pass; ++i) {
		if (!on[i]) continue;
		const ChunkPass& p = P.pass[i];
		const AttnChunkArgs b = pass_args(p);
		const dim3 grid((unsigned)p.workers, (unsigned)((p.R + 31) / 32));
		INF_TRY(launch_pdl(kv->dtype == InfBF16 ? k_attn_chunk_combine<bf16> : k_attn_chunk_combine<float>, grid, dim3(kAcCombineThreads),
		                   0, st, b));
	}
	return Success;
}

} // extern "C"
