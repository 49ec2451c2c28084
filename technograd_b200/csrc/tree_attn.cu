// tree_attn.cu -- attention of drafted tokens over a paged cache, and the attention weight
// that the cache's positions receive.
#include "paged.cuh"

namespace tgc {

struct AttnArgs {
	PgCache c;
	PgDrafts d;
	char *out;
	long long out_seq, out_tok, out_head; // bytes
	float *lse;
};

// One warp's dot product of q (in registers, lane's elements i * 32 + lane) with a row.
template <class T, int N>
__device__ __forceinline__ float warp_dot(const float (&q)[N], const char *row, int dim, int lane)
{
	float s = 0;
#pragma unroll
	for (int i = 0; i < N; i++)
		if (i * 32 + lane < dim) s += q[i] * PgElem<T>::get(((const T *)row)[i * 32 + lane]);
#pragma unroll
	for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
	return s;
}

// One CTA per (query row, sequence): its four warps take the keys in turn, a key at a time, each
// with a running maximum m and sum l of exp(s - m); the warps' parts are joined at the end.
template <class T>
__global__ void __launch_bounds__(128) k_tree_attn(const AttnArgs p)
{
	constexpr int N = 8; // 256 elements of a row over 32 lanes
	__shared__ float sm[4], sl[4], so[4][256];
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = p.c.dim;
	long long r = blockIdx.x;
	const int j = (int)(r % p.d.nq), h = j / p.d.group;
	r /= p.d.nq;
	const int t = (int)(r % p.d.tokens), b = (int)(r / p.d.tokens);
	const int n = p.c.length(b), cnt = p.d.drafted(b);
	const bool live = t < cnt;
	const unsigned long long see = live ? p.d.sees(b, t, cnt) : 0;
	float q[N], o[N], m = -INFINITY, l = 0;
#pragma unroll
	for (int i = 0; i < N; i++) {
		const int x = i * 32 + lane;
		q[i] = x < dim ? PgElem<T>::get(((const T *)(p.d.q + b * p.d.q_seq + t * p.d.q_tok + j * p.d.q_head))[x]) : 0;
		o[i] = 0;
	}
	const int *tab = p.c.table + (long long)b * p.c.cols;
	for (long long x = warp; live && x < (long long)n + cnt; x += 4) {
		const char *kr, *vr;
		if (x < n) {
			const long long at = p.c.row(tab, (int)x);
			kr = at < 0 ? nullptr : p.c.k + at + h * p.c.head_b;
			vr = at < 0 ? nullptr : p.c.v + at + h * p.c.head_b;
		} else {
			if (!(see >> (x - n) & 1)) continue;
			kr = p.d.k + b * p.d.kv_seq + (x - n) * p.d.kv_tok + h * p.d.kv_head;
			vr = p.d.v + b * p.d.kv_seq + (x - n) * p.d.kv_tok + h * p.d.kv_head;
		}
		const float s = kr ? warp_dot<T>(q, kr, dim, lane) * p.d.scale : 0;
		if (s == -INFINITY) continue;
		const float m2 = fmaxf(m, s), a = expf(m - m2), e = expf(s - m2);
		l = l * a + e;
#pragma unroll
		for (int i = 0; i < N; i++) {
			const int y = i * 32 + lane;
			o[i] = o[i] * a + (vr && y < dim ? e * PgElem<T>::get(((const T *)vr)[y]) : 0);
		}
		m = m2;
	}
	if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
	for (int i = 0; i < N; i++) so[warp][i * 32 + lane] = o[i];
	__syncthreads();
	m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
	l = 0;
	float a[4];
	for (int w = 0; w < 4; w++) {
		a[w] = sm[w] == -INFINITY ? 0 : expf(sm[w] - m);
		l += sl[w] * a[w];
	}
	for (int x = threadIdx.x; x < dim; x += 128) {
		float v = 0;
		for (int w = 0; w < 4; w++) v += so[w][x] * a[w];
		((T *)(p.out + b * p.out_seq + t * p.out_tok + j * p.out_head))[x] = PgElem<T>::put(l == 0 ? 0 : v / l);
	}
	if (threadIdx.x == 0) p.lse[blockIdx.x] = l == 0 ? -INFINITY : m + logf(l);
}

struct WeightArgs {
	PgCache c;
	PgDrafts d;
	const float *lse;
	const unsigned long long *select;
	const float *acc;
	long long acc_seq, acc_head;
	float *acc_out, *fresh;
	int chunks; // key chunks per (sequence, kv head)
};

// One CTA per (sequence, kv head, 64 positions), a warp per position: the rows of q are dotted
// with the position's key one after the other. The drafted tokens follow the last cached chunk.
template <class T>
__global__ void __launch_bounds__(128) k_attn_weights(const WeightArgs p)
{
	constexpr int N = 8;
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = p.c.dim;
	long long r = blockIdx.x;
	const int chunk = (int)(r % p.chunks);
	r /= p.chunks;
	const int h = (int)(r % p.c.nkv), b = (int)(r / p.c.nkv);
	const int n = p.c.length(b), cnt = p.d.drafted(b);
	const unsigned long long sel = p.select ? p.select[b] : ~0ull;
	const int *tab = p.c.table + (long long)b * p.c.cols;
	const bool last = chunk == p.chunks - 1;
	const int to = last ? p.d.tokens : min(64, p.c.max_len - chunk * 64);
	for (int i = warp; i < to; i += 4) {
		const int x = chunk * 64 + i; // cached position, or drafted token i
		const bool there = last ? i < cnt : x < n;
		const char *kr = nullptr;
		if (last) kr = p.d.k + b * p.d.kv_seq + i * p.d.kv_tok + h * p.d.kv_head;
		else if (there) {
			const long long at = p.c.row(tab, x);
			kr = at < 0 ? nullptr : p.c.k + at + h * p.c.head_b;
		}
		float k[N], w = 0;
#pragma unroll
		for (int y = 0; y < N; y++) k[y] = there && kr && y * 32 + lane < dim ? PgElem<T>::get(((const T *)kr)[y * 32 + lane]) : 0;
		for (int t = 0; there && t < cnt; t++) {
			if (!(sel >> t & 1) || (last && !(p.d.sees(b, t, cnt) >> i & 1))) continue;
			for (int g = 0; g < p.d.group; g++) {
				const int j = h * p.d.group + g;
				const float lse = p.lse[((long long)b * p.d.tokens + t) * p.d.nq + j];
				if (lse == -INFINITY) continue;
				w += expf(warp_dot<T>(k, p.d.q + b * p.d.q_seq + t * p.d.q_tok + j * p.d.q_head, dim, lane) * p.d.scale - lse);
			}
		}
		if (lane) continue;
		if (last) p.fresh[((long long)b * p.c.nkv + h) * p.d.tokens + i] = w;
		else
			p.acc_out[((long long)b * p.c.nkv + h) * p.c.max_len + x] =
				there ? (p.acc ? p.acc[b * p.acc_seq + h * p.acc_head + x] : 0) + w : 0;
	}
}

} // namespace tgc

using namespace tgc;

extern "C" long long tg_cuda_tree_attn_workspace(const tg_cuda_kv *c, const tg_cuda_drafts *d)
{
	clear_err();
	PgCache pc;
	PgDrafts pd;
	int rc = pg_cache("tg_cuda_tree_attn_workspace", c, &pc);
	if (rc || (rc = pg_drafts("tg_cuda_tree_attn_workspace", c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &pd))) return rc;
	return 0;
}

extern "C" int tg_cuda_tree_attn(const tg_cuda_kv *c, const tg_cuda_drafts *d, void *out, long long out_seq, long long out_tok,
				 long long out_head, float *lse, void *work, long long work_bytes, void *stream)
{
	const char *who = "tg_cuda_tree_attn";
	clear_err();
	AttnArgs p = {};
	int rc, sms;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K | PG_USE_V, 64, &p.d))) return rc;
	const int e = pg_size(c->type);
	if (c->seqs && (!out || !lse)) return set_err(TG_CUDA_EINVAL, "%s: NULL output", who);
	if (((uintptr_t)out & 15) || ((out_seq | out_tok | out_head) * e & 15))
		return set_err(TG_CUDA_EINVAL, "%s: out rows must start on 16-byte boundaries", who);
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0) return rc;
	p.out = (char *)out, p.out_seq = out_seq * e, p.out_tok = out_tok * e, p.out_head = out_head * e, p.lse = lse;
	const long long blocks = (long long)c->seqs * d->tokens * d->nq;
	if (blocks > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of %d tokens and %d heads", who, c->seqs, d->tokens, d->nq);
	cudaStream_t st = (cudaStream_t)stream;
	if (c->type == TG_CUDA_F32) k_tree_attn<float><<<(unsigned)blocks, 128, 0, st>>>(p);
	else if (c->type == TG_CUDA_F16) k_tree_attn<__half><<<(unsigned)blocks, 128, 0, st>>>(p);
	else k_tree_attn<__nv_bfloat16><<<(unsigned)blocks, 128, 0, st>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

extern "C" int tg_cuda_attn_weights(const tg_cuda_kv *c, const tg_cuda_drafts *d, const float *lse, const unsigned long long *select,
				    const float *acc, long long acc_seq, long long acc_head, float *acc_out, float *fresh, void *stream)
{
	const char *who = "tg_cuda_attn_weights";
	clear_err();
	WeightArgs p = {};
	int rc, sms;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K, 64, &p.d))) return rc;
	if (c->seqs && (!lse || !fresh || (!acc_out && c->max_len))) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (acc && acc == acc_out && (acc_head != c->max_len || acc_seq != (long long)c->nkv * c->max_len))
		return set_err(TG_CUDA_EINVAL, "%s: acc may be acc_out with acc_out's own strides only", who);
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0) return rc;
	p.lse = lse, p.select = select, p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head, p.acc_out = acc_out, p.fresh = fresh;
	p.chunks = (c->max_len + 63) / 64 + 1;
	const long long blocks = (long long)c->seqs * c->nkv * p.chunks;
	if (blocks > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of up to %d positions", who, c->seqs, c->max_len);
	cudaStream_t st = (cudaStream_t)stream;
	if (c->type == TG_CUDA_F32) k_attn_weights<float><<<(unsigned)blocks, 128, 0, st>>>(p);
	else if (c->type == TG_CUDA_F16) k_attn_weights<__half><<<(unsigned)blocks, 128, 0, st>>>(p);
	else k_attn_weights<__nv_bfloat16><<<(unsigned)blocks, 128, 0, st>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}
