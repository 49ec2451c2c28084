// evict.cu -- tg_cuda_kv_evict: the positions of a paged cache to keep by their accumulated
// attention weight, and their rows' copy to other pages.
#include <cooperative_groups.h>

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
	int pieces, lg;   // 16-byte pieces of a row's K and V together, and its logarithm where it is a power of two, else -1
	long long heads;  // sequences times kv heads
	int fused;        // the selecting CTA copies its rows itself
};

// A weight's place in the order: unsigned, larger = kept first. Negative numbers reverse, -0 is 0,
// NaN (1) is below -infinity (whose key is 0x007fffff). EV_NONE is a position that does not compete.
constexpr uint32_t EV_NONE = 0;
__device__ __forceinline__ uint32_t evict_key(float x)
{
	if (isnan(x)) return 1;
	const uint32_t u = __float_as_uint(x == 0 ? 0.0f : x);
	return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The weight of a key (a zero is +0, a NaN any).
__device__ __forceinline__ float evict_weight(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The copy, bound by HBM: a warp takes 32 kept positions of a head; a lane finds the places of one of them,
// then the warp moves the rows' 16-byte pieces, K and V, eight loads in flight a lane. Measured: 4000 rows of 256 bytes
// for each of those heads 116 us, 5.6 TB/s read and written.
__device__ __forceinline__ void evict_copy32(const EvictArgs &p, long long bh, int group)
{
	const int lane = threadIdx.x & 31, i = group * 32 + lane, h = (int)(bh % p.src.nkv);
	const long long b = bh / p.src.nkv;
	const int from = i < p.budget ? p.keep[bh * p.budget + i] : -1;
	uint32_t s = PG_NONE, t = PG_NONE; // places, PG_NONE: zeros; no copy
	if (from >= 0) {
		if (i >= (long long)p.dst.page * p.dst.cols) p.dst.report(PG_ROOM);
		else {
			const int a = from / p.src.page, d = i / p.dst.page;
			t = p.dst.at(p.dst.table[b * p.dst.cols + d], i - d * p.dst.page);
			s = p.src.at(p.src.table[b * p.src.cols + a], from - a * p.src.page);
		}
	}
	const int rows = 32 - __clz(__ballot_sync(~0u, t != PG_NONE)), pieces = p.pieces, half = pieces / 2;
	const char *sk = p.src.k + h * p.src.head_b, *sv = p.src.v + h * p.src.head_b;
	char *tk = p.dst.k + h * p.dst.head_b, *tv = p.dst.v + h * p.dst.head_b;
	for (int x0 = 0; x0 < rows * pieces; x0 += 32 * 8) {
		uint4 v[8];
		char *to[8];
#pragma unroll
		for (int u = 0; u < 8; u++) {
			const int x = x0 + u * 32 + lane, row = p.lg >= 0 ? x >> p.lg : x / pieces, c = x - row * pieces;
			const uint32_t a = __shfl_sync(~0u, s, row & 31), d = __shfl_sync(~0u, t, row & 31);
			const int o = (c < half ? c : c - half) * 16;
			to[u] = row < rows && d != PG_NONE ? (c < half ? tk : tv) + ((unsigned long long)d << p.dst.shift) + o : nullptr;
			v[u] = make_uint4(0, 0, 0, 0);
			if (to[u] && a != PG_NONE) v[u] = __ldcs((const uint4 *)((c < half ? sk : sv) + ((unsigned long long)a << p.src.shift) + o));
		}
#pragma unroll
		for (int u = 0; u < 8; u++)
			if (to[u]) *(uint4 *)to[u] = v[u];
	}
}

__global__ void __launch_bounds__(256) k_evict_copy(const EvictArgs p)
{
	pdl_launch();
	pdl_wait();
	const int groups = (p.budget + 31) / 32;
	const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), bh = w / groups;
	if (bh < p.heads) evict_copy32(p, bh, (int)(w - bh * groups));
}

constexpr int EV_THREADS = 1024, EV_WARPS = EV_THREADS / 32, EV_CLUSTER = 8, EV_LIST = 512;
constexpr long long EV_FUSED = 128 * 1024; // bytes of a head's kept rows

// What the CTAs of a cluster exchange.
struct EvictShared {
	int part[2][EV_WARPS];    // a warp's counts
	int count[2][EV_CLUSTER]; // the CTAs' counts, in turns
	int sure[EV_CLUSTER], ties[EV_CLUSTER];
	uint32_t thr;
	int above, least, n_list;
	uint32_t list[EV_LIST];
};

// One cluster of CTAs per (sequence, kv head). A CTA has an equal run of the positions, a warp a run of that
// one, and a thread holds KPT of their keys in registers (0: any number, read again from L2 each time).
// The threshold is the want-th largest key, found bit by bit: count the keys that reach a candidate, over
// the cluster. Once few enough keys share the threshold's prefix (after about ten bits),
// the first CTA's first warp finishes alone on their list. Every position above the threshold is kept, and the first
// ones that equal it; ballots over the runs give each its place.
// What bounds it: latency. The weights come in one round of loads, a count is 2 KPT instructions a
// thread and a barrier or two. Measured: 192 heads of up to 32001 positions 63 us, two CTAs after each other on an SM.
template <int KPT>
__device__ __forceinline__ void evict_select(const EvictArgs &p, EvictShared &s)
{
	namespace cg = cooperative_groups;
	cg::cluster_group cluster = cg::this_cluster();
	const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
	const long long head = blockIdx.x / ranks;
	const int h = (int)(head % p.src.nkv), b = (int)(head / p.src.nkv), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	const int n = p.src.length(b);
	const float *acc = p.acc + b * p.acc_seq + h * p.acc_head;
	int *keep = p.keep + head * p.budget;
	float *out = p.acc_out + head * p.budget;
	const int kept = min(n, p.budget), all = ranks * EV_THREADS, me = rank * EV_THREADS + tid;
	if (h == 0 && me == 0) p.len_out[b] = kept;
	for (int i = kept + me; i < p.budget; i += all) keep[i] = -1, out[i] = 0;
	if (n <= p.budget) { // of the whole cluster
		for (int i = me; i < n; i += all) keep[i] = i, out[i] = acc[i];
		return;
	}
	// the first and last positions have their places; want of those between compete for theirs
	const int lo = p.sink, hi = n - p.recent, want = p.budget - p.sink - p.recent; // 0 <= want < hi - lo
	for (int i = me; i < lo; i += all) keep[i] = i, out[i] = acc[i];
	for (int i = hi + me; i < n; i += all) keep[i - n + p.budget] = i, out[i - n + p.budget] = acc[i];
	if (want == 0) return; // of the whole cluster
	if (ranks > 1) cluster.barrier_arrive(); // a CTA's shared memory may be written to once the CTA has begun: waited for after the loads below
	keep += lo, out += lo;
	// the warp's positions, `per` from w0 on: all whole warps' worth
	const int per = (int)(((long long)n + ranks * EV_WARPS * 32 - 1) / (ranks * EV_WARPS * 32)) * 32; // at most 32 KPT
	const int w0 = (rank * EV_WARPS + warp) * per; // within int: at most 8192 past n
	auto fresh = [&](int i) { // (every lane loads, so that the loads go out together)
		const uint32_t x = evict_key(acc[min(i, n - 1)]);
		return i < lo || i >= hi ? EV_NONE : x;
	};
	uint32_t k[KPT ? KPT : 1];
	if constexpr (KPT > 0) {
		float a[KPT];
#pragma unroll
		for (int u = 0; u < KPT; u++) a[u] = acc[min(w0 + u * 32 + lane, n - 1)];
#pragma unroll
		for (int u = 0; u < KPT; u++) {
			const int i = w0 + u * 32 + lane;
			k[u] = i < lo || i >= hi || u * 32 >= per ? EV_NONE : evict_key(a[u]);
		}
	}
	if (ranks > 1) cluster.barrier_wait();
	// f(position, key) for the thread's positions, in order, the warp's lanes together
	auto each = [&](auto f) {
		if constexpr (KPT > 0) {
#pragma unroll
			for (int u = 0; u < KPT; u++) f(w0 + u * 32 + lane, k[u]); // (past per: no keys; a branch here costs more than they do)
		} else
			for (int i = w0; i < w0 + per && i < n; i += 32) f(i + lane, fresh(i + lane));
	};
	auto sync = [&]() {
		if (ranks > 1) cluster.sync();
		else __syncthreads();
	};
	int turn = 0;
	// the cluster's total of a count, to every thread of it
	auto total = [&](int v) {
		v = __reduce_add_sync(~0u, v);
		if (lane == 0) s.part[turn][warp] = v;
		__syncthreads();
		v = __reduce_add_sync(~0u, s.part[turn][lane]);
		if (ranks > 1) {
			if (tid < ranks) *cluster.map_shared_rank(&s.count[turn][rank], tid) = v;
			cluster.sync();
			v = 0;
			for (int r = 0; r < ranks; r++) v += s.count[turn][r];
		}
		turn ^= 1; // the next count's words are read by nobody any more
		return v;
	};
	auto reach = [&](uint32_t c) { // keys >= c, this thread's
		int m = 0;
		each([&](int, uint32_t x) { m += x >= c; });
		return m;
	};
	uint32_t thr = 0;        // its bits so far
	int bit = 31, above = 0, least = hi - lo; // keys above every one that shares thr's bits; keys that reach thr, at most
	auto step = [&]() {
		const uint32_t c = thr | 1u << bit;
		const int m = total(reach(c));
		if (m >= want) thr = c, least = m;
		else above = m;
		bit--;
	};
	// the last bits of thr, by the first warp alone: c keys on its list
	auto finish = [&](int c) {
		uint32_t x[EV_LIST / 32];
#pragma unroll
		for (int u = 0; u < EV_LIST / 32; u++) x[u] = u * 32 + lane < c ? s.list[u * 32 + lane] : EV_NONE;
		auto those = [&](uint32_t from) {
			int m = 0;
#pragma unroll
			for (int u = 0; u < EV_LIST / 32; u++) m += x[u] >= from;
			return above + __reduce_add_sync(~0u, m);
		};
		for (; bit >= 0; bit--)
			if (those(thr | 1u << bit) >= want) thr |= 1u << bit;
		least = those(thr);
		above = those(thr + 1);
		if (lane == 0) s.thr = thr, s.above = above, s.least = least;
	};
	if (KPT == 1 && ranks == 1 && n <= EV_LIST) { // all on the list at once
		if (tid < EV_LIST) s.list[tid] = fresh(tid);
		__syncthreads();
		if (warp == 0) finish(n);
		__syncthreads();
		thr = s.thr, above = s.above, least = s.least;
	} else {
		while (bit >= 0 && least - above > EV_LIST) step();
		if (bit >= 0) {
			// the keys that share the prefix, on the first CTA's list
			if (rank == 0 && tid == 0) s.n_list = 0;
			sync();
			const uint32_t end = thr + (2u << bit) - 1; // the last key with the prefix
			EvictShared *first = ranks > 1 ? cluster.map_shared_rank(&s, 0) : &s;
			each([&](int, uint32_t x) {
				if (x >= thr && x <= end && x != EV_NONE) first->list[atomicAdd(&first->n_list, 1)] = x; // any order: only counts are taken of it
			});
			sync();
			if (rank == 0 && warp == 0) finish(s.n_list);
			sync();
			thr = first->thr, above = first->above, least = first->least;
		} else above = total(reach(thr + 1));
	}
	int ties = want - above; // of the positions that equal thr, the first so many
	if (least == want) thr--, ties = 0; // all of them
	// ---- in order: counts of each warp's run, then each writes its own
	int n_sure = 0, n_tie = 0;
	each([&](int, uint32_t x) {
		n_sure += x > thr;
		if (ties) n_tie += x == thr;
	});
	n_sure = __reduce_add_sync(~0u, n_sure), n_tie = __reduce_add_sync(~0u, n_tie);
	__syncthreads();
	if (lane == 0) s.part[0][warp] = n_sure, s.part[1][warp] = n_tie;
	__syncthreads();
	const int ps = s.part[0][lane], pt = s.part[1][lane];
	int done = __reduce_add_sync(~0u, lane < warp ? ps : 0), tied = __reduce_add_sync(~0u, lane < warp ? pt : 0);
	if (ranks > 1) {
		const int as = __reduce_add_sync(~0u, ps), at = __reduce_add_sync(~0u, pt);
		if (tid < ranks) {
			EvictShared *o = cluster.map_shared_rank(&s, tid);
			o->sure[rank] = as, o->ties[rank] = at;
		}
		cluster.sync();
		for (int r = 0; r < rank; r++) done += s.sure[r], tied += s.ties[r];
	}
	done += min(tied, ties);
	const unsigned below = (1u << lane) - 1;
	each([&](int i, uint32_t x) {
		bool take = x > thr;
		if (ties) { // the first `ties` of those that equal the threshold
			const bool t = x == thr;
			const unsigned bt = __ballot_sync(~0u, t);
			take |= t && tied + __popc(bt & below) < ties;
			tied += __popc(bt);
		}
		const unsigned bk = __ballot_sync(~0u, take);
		if (take) {
			const int at = done + __popc(bk & below);
			keep[at] = i, out[at] = evict_weight(x); // (a load here would wait for the stores of the step before)
		}
		done += __popc(bk);
	});
}

template <int KPT>
__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const EvictArgs p)
{
	__shared__ EvictShared s;
	pdl_launch();
	pdl_wait();
	evict_select<KPT>(p, s);
	if (!p.fused) return;
	__syncthreads(); // the CTA's kept positions are written
	for (int g = threadIdx.x >> 5; g < (p.budget + 31) / 32; g += EV_WARPS) evict_copy32(p, blockIdx.x, g);
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
	if ((rc = pg_apart(who, "the destination", to.head_dim, {to.page_stride, to.head_stride, to.pos_stride}, {to.pages, to.nkv, to.page}))) return rc;
	if (budget <= 0 || recent < 0 || sink < 0 || recent > budget - sink)
		return set_err(TG_CUDA_EINVAL, "%s: budget %d, recent %d, sink %d", who, budget, recent, sink);
	if (src->seqs && (!keep || !acc_out || !len_out || (!acc && src->max_len))) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (((uintptr_t)acc | (uintptr_t)keep | (uintptr_t)acc_out | (uintptr_t)len_out) & 3) return set_err(TG_CUDA_EINVAL, "%s: a pointer is not on a 4-byte boundary", who);
	if ((acc_seq < 0 && src->seqs > 1) || (acc_head < 0 && src->nkv > 1)) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	if (len_out == src->len && src->seqs) return set_err(TG_CUDA_EINVAL, "%s: len_out may not be the cache's len", who);
	if ((rc = pg_device(who, &sms, &p.src.status)) || src->seqs == 0) return rc;
	p.dst.status = p.src.status;
	p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head, p.budget = budget, p.recent = recent, p.sink = sink;
	p.keep = keep, p.acc_out = acc_out, p.len_out = len_out, p.pieces = src->head_dim * pg_size(src->type) / 8;
	p.lg = -1;
	if (!(p.pieces & (p.pieces - 1)))
		for (p.lg = 0; 1 << p.lg < p.pieces;) p.lg++;
	p.heads = (long long)src->seqs * src->nkv;
	const long long blocks = (p.heads * ((budget + 31ll) / 32) + 7) / 8;
	if (blocks > 0x7fffffff || p.heads * EV_CLUSTER > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences, budget %d", who, src->seqs, budget);
	// a head's CTAs: as many as hold its keys in registers, and more where heads are fewer than SMs and the runs stay of
	// some length (below 4096 keys a cluster's barriers cost more than the shorter passes give)
	int ranks = 1;
	while (ranks < EV_CLUSTER && (src->max_len > 32ll * EV_THREADS * ranks || (p.heads * ranks * 2 <= sms && src->max_len > 4096 * 2 * ranks))) ranks *= 2;
	const long long run = ((long long)src->max_len + ranks - 1) / ranks;
	// little to copy: a second kernel would take longer than the selecting CTAs do (200 positions of 64 bytes: 15 us a call against 12)
	p.fused = ranks == 1 && p.heads <= sms && (long long)budget * p.pieces * 16 <= EV_FUSED;
	cudaStream_t st = (cudaStream_t)stream;
	cudaLaunchConfig_t cfg = {};
	cudaLaunchAttribute attr[2];
	cfg.gridDim = dim3((unsigned)(p.heads * ranks)), cfg.blockDim = dim3(EV_THREADS), cfg.stream = st;
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
	attr[1].id = cudaLaunchAttributeClusterDimension, attr[1].val.clusterDim.x = ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
	cfg.attrs = attr, cfg.numAttrs = ranks > 1 ? 2 : 1;
	TGC_CUDA(cudaLaunchKernelEx(&cfg, run <= EV_THREADS ? k_evict_select<1> : run <= 8 * EV_THREADS ? k_evict_select<8> : run <= 16 * EV_THREADS ? k_evict_select<16> : run <= 32 * EV_THREADS ? k_evict_select<32> : k_evict_select<0>, p));
	if (!p.fused) TGC_CUDA(launch_pdl(k_evict_copy, dim3((unsigned)blocks), dim3(256), 0, st, p));
	return TG_CUDA_OK;
}
