// evict.cu -- tg_cuda_kv_evict: the positions of a paged cache to keep by their accumulated
// attention weight, and their rows' copy to other pages.
#include "paged.cuh"

namespace tgc {

struct EvictArgs {
	PgCache src, dst;
	const float *acc;
	long long acc_seq, acc_head;
	int budget, recent, sink;
	int *keep;
	float *acc_out;
	int *len_out;
	int chunks; // 16-byte pieces of a row
	long long heads; // sequences times kv heads
};

// A weight's place in the order: unsigned, larger = kept first. Negative numbers reverse, -0 is 0,
// NaN is below -infinity (whose key is 0x007fffff).
__device__ __forceinline__ uint32_t evict_key(float x)
{
	if (isnan(x)) return 0;
	const uint32_t u = __float_as_uint(x == 0 ? 0.0f : x);
	return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the CTA's 1024 threads, to every thread.
__device__ __forceinline__ int block_sum(int v, int *s)
{
	v = __reduce_add_sync(~0u, v);
	__syncthreads();
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	return __reduce_add_sync(~0u, s[threadIdx.x & 31]);
}

// One CTA per (sequence, kv head): the threshold key by bisection over its 32 bits, then one pass
// in order that takes every position above it and the first ones that equal it.
__global__ void __launch_bounds__(1024) k_evict_select(const EvictArgs p)
{
	__shared__ int s[32], sa[32], sb[32];
	const int h = blockIdx.x % p.src.nkv, b = blockIdx.x / p.src.nkv, tid = threadIdx.x;
	const int n = p.src.length(b);
	const float *acc = p.acc + b * p.acc_seq + h * p.acc_head;
	int *keep = p.keep + (long long)blockIdx.x * p.budget;
	float *out = p.acc_out + (long long)blockIdx.x * p.budget;
	const int kept = min(n, p.budget);
	if (h == 0 && tid == 0) p.len_out[b] = kept;
	for (int i = kept + tid; i < p.budget; i += 1024) keep[i] = -1, out[i] = 0;
	if (n <= p.budget) {
		for (int i = tid; i < n; i += 1024) keep[i] = i, out[i] = acc[i];
		return;
	}
	const int lo = p.sink, hi = n - p.recent, want = p.budget - p.sink - p.recent; // 0 <= want < hi - lo
	uint32_t thr = 0;                                                             // the want-th largest key
	for (int bit = 31; bit >= 0; bit--) {
		const uint32_t c = thr | 1u << bit;
		int m = 0;
		for (int i = lo + tid; i < hi; i += 1024) m += evict_key(acc[i]) >= c;
		if (block_sum(m, s) >= want) thr = c;
	}
	int above = 0;
	for (int i = lo + tid; i < hi; i += 1024) above += evict_key(acc[i]) > thr;
	int ties = want - block_sum(above, s); // of the positions equal to thr, the first so many
	if (want == 0) thr = 0xffffffffu, ties = 0;
	int done = 0, tied = 0;
	for (int i0 = 0; i0 < n; i0 += 1024) {
		const int i = i0 + tid;
		const bool mid = i >= lo && i < hi;
		const uint32_t k = mid ? evict_key(acc[i]) : 0;
		const bool tie = mid && k == thr, sure = i < n && (!mid || k > thr);
		const unsigned bt = __ballot_sync(~0u, tie), below = (1u << (tid & 31)) - 1;
		__syncthreads();
		if ((tid & 31) == 0) sa[tid >> 5] = __popc(bt);
		__syncthreads();
		int rank = tied + __popc(bt & below);
		for (int w = 0; w < 32; w++) {
			if (w < tid >> 5) rank += sa[w];
			tied += sa[w];
		}
		const bool take = sure || (tie && rank < ties);
		const unsigned bk = __ballot_sync(~0u, take);
		if ((tid & 31) == 0) sb[tid >> 5] = __popc(bk);
		__syncthreads();
		int at = done + __popc(bk & below);
		for (int w = 0; w < 32; w++) {
			if (w < tid >> 5) at += sb[w];
			done += sb[w];
		}
		if (take) keep[at] = i, out[at] = acc[i];
	}
}

// One warp per (kept position, kv head, sequence): the row's 16-byte pieces of K, then of V.
__global__ void __launch_bounds__(256) k_evict_copy(const EvictArgs p)
{
	const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
	const int lane = threadIdx.x & 31;
	const long long bh = w / p.budget;
	const int i = (int)(w - bh * p.budget), h = (int)(bh % p.src.nkv);
	const long long b = bh / p.src.nkv;
	if (bh >= p.heads) return;
	const int from = p.keep[bh * p.budget + i];
	if (from < 0) return;
	if (i >= (long long)p.dst.page * p.dst.cols) {
		if (lane == 0) p.dst.report(PG_ROOM);
		return;
	}
	const long long s = p.src.row(p.src.table + b * p.src.cols, from), t = p.dst.row(p.dst.table + b * p.dst.cols, i);
	if (t < 0) return;
	for (int x = lane; x < 2 * p.chunks; x += 32) {
		const int o = (x < p.chunks ? x : x - p.chunks) * 16;
		const char *a = (x < p.chunks ? p.src.k : p.src.v) + s + h * p.src.head_b + o;
		*(uint4 *)((x < p.chunks ? p.dst.k : p.dst.v) + t + h * p.dst.head_b + o) = s < 0 ? make_uint4(0, 0, 0, 0) : *(const uint4 *)a;
	}
}

} // namespace tgc

using namespace tgc;

extern "C" int tg_cuda_kv_evict(const tg_cuda_kv *src, const tg_cuda_kv *dst, const float *acc, long long acc_seq, long long acc_head,
				int budget, int recent, int sink, int *keep, float *acc_out, int *len_out, void *stream)
{
	const char *who = "tg_cuda_kv_evict";
	clear_err();
	EvictArgs p = {};
	int rc, sms;
	if (!dst) return set_err(TG_CUDA_EINVAL, "%s: NULL cache", who);
	tg_cuda_kv to = *dst;
	to.len = src ? src->len : nullptr, to.max_len = 0; // not read
	if ((rc = pg_cache(who, src, &p.src)) || (rc = pg_cache(who, &to, &p.dst))) return rc;
	if (to.type != src->type || to.seqs != src->seqs || to.nkv != src->nkv || to.head_dim != src->head_dim)
		return set_err(TG_CUDA_EINVAL, "%s: the destination's type, seqs, nkv or head_dim differ", who);
	if (budget <= 0 || recent < 0 || sink < 0 || recent > budget - sink)
		return set_err(TG_CUDA_EINVAL, "%s: budget %d, recent %d, sink %d", who, budget, recent, sink);
	if (src->seqs && (!keep || !acc_out || !len_out || (!acc && src->max_len))) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (len_out == src->len && src->seqs) return set_err(TG_CUDA_EINVAL, "%s: len_out may not be the cache's len", who);
	if ((rc = pg_device(who, &sms, &p.src.status)) || src->seqs == 0) return rc;
	p.dst.status = p.src.status;
	p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head, p.budget = budget, p.recent = recent, p.sink = sink;
	p.keep = keep, p.acc_out = acc_out, p.len_out = len_out, p.chunks = src->head_dim * pg_size(src->type) / 16;
	const long long heads = (long long)src->seqs * src->nkv, blocks = (heads * budget + 7) / 8;
	p.heads = heads;
	if (blocks > 0x7fffffff || heads > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences, budget %d", who, src->seqs, budget);
	cudaStream_t st = (cudaStream_t)stream;
	k_evict_select<<<(unsigned)heads, 1024, 0, st>>>(p);
	TGC_LAUNCH_CHECK();
	k_evict_copy<<<(unsigned)blocks, 256, 0, st>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}
