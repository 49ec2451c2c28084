// paged.cu -- descriptions of a paged key/value cache, checked on the host, and
// tg_cuda_kv_commit.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <utility>

#include "paged.cuh"

namespace tgc {

constexpr int PG_DEVICES = 64;
static std::mutex g_pg_mu;
static struct { int sms; int *host, *dev; } g_pg[PG_DEVICES];

int pg_sms(const char *who, int *dev, int *sms)
{
	cudaError_t e = cudaGetDevice(dev);
	if (e != cudaSuccess) return set_err(TG_CUDA_ENODEV, "%s: cudaGetDevice: %s", who, cudaGetErrorString(e));
	if (*dev < 0 || *dev >= PG_DEVICES) return set_err(TG_CUDA_EINVAL, "%s: device ordinal %d", who, *dev);
	std::lock_guard<std::mutex> lk(g_pg_mu);
	auto &g = g_pg[*dev];
	if (!g.sms) {
		int n = 0;
		TGC_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev));
		g.sms = n;
	}
	*sms = g.sms;
	return TG_CUDA_OK;
}

int pg_device(const char *who, int *sms, int **status)
{
	int dev = -1, rc = pg_sms(who, &dev, sms);
	if (rc) return rc;
	std::lock_guard<std::mutex> lk(g_pg_mu);
	auto &g = g_pg[dev];
	if (!g.host) {
		int *h = nullptr;
		TGC_CUDA(cudaHostAlloc((void **)&h, PG_WORDS * sizeof(int), cudaHostAllocMapped));
		for (int i = 0; i < PG_WORDS; i++) h[i] = 0;
		cudaError_t e = cudaHostGetDevicePointer((void **)&g.dev, h, 0);
		if (e != cudaSuccess) {
			cudaFreeHost(h);
			return set_err(TG_CUDA_ECUDA, "%s: cudaHostGetDevicePointer: %s", who, cudaGetErrorString(e));
		}
		g.host = h;
	}
	int met[PG_WORDS], any = 0;
	for (int i = 0; i < PG_WORDS; i++) any |= met[i] = __atomic_exchange_n(g.host + i, 0, __ATOMIC_ACQ_REL);
	if (any)
		return set_err(TG_CUDA_EDEVICE, "%s: an earlier call on this device met%s%s%s%s%s%s", who,
			       met[PG_LEN] ? " a len outside [0, max_len];" : "", met[PG_PAGE] ? " a page number outside the pool;" : "",
			       met[PG_PATH] ? " a path entry outside the drafted tokens;" : "",
			       met[PG_ROOM] ? " a row past the table or the weights;" : "", met[PG_WAIT] ? " a wait that timed out;" : "",
			       met[PG_GROUP] ? " a group of sequences or a shared length that does not suit;" : "");
	*status = g.dev;
	return TG_CUDA_OK;
}

// A stride along one element alone is never used, and need not suit
static long long pg_stride(long long s, int n, int e) { return n <= 1 && (s < 0 || s * e & 15) ? 0 : s; }

int pg_cache(const char *who, const tg_cuda_kv *desc, PgCache *o)
{
	if (!desc) return set_err(TG_CUDA_EINVAL, "%s: NULL cache", who);
	tg_cuda_kv copy = *desc, *c = &copy;
	if (c->type != TG_CUDA_F32 && c->type != TG_CUDA_F16 && c->type != TG_CUDA_BF16)
		return set_err(TG_CUDA_EINVAL, "%s: element type %d", who, c->type);
	const int e = pg_size(c->type);
	if (c->seqs < 0 || c->nkv <= 0 || c->page <= 0 || c->pages < 0 || c->table_cols < 0 || c->max_len < 0)
		return set_err(TG_CUDA_EINVAL, "%s: bad cache (seqs %d nkv %d page %d pages %d table_cols %d max_len %d)", who, c->seqs, c->nkv,
			       c->page, c->pages, c->table_cols, c->max_len);
	if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim * e % 16)
		return set_err(TG_CUDA_EINVAL, "%s: head_dim %d: at most 256, in rows of a multiple of 16 bytes", who, c->head_dim);
	if (c->max_len > (long long)c->page * c->table_cols)
		return set_err(TG_CUDA_EINVAL, "%s: max_len %d is more than %d pages of %d hold", who, c->max_len, c->table_cols, c->page);
	if (c->max_len > 0x7fff0000) return set_err(TG_CUDA_EINVAL, "%s: max_len %d", who, c->max_len);
	if (c->seqs && (!c->len || (!c->table && c->table_cols > 0) || ((!c->k || !c->v) && c->pages > 0)))
		return set_err(TG_CUDA_EINVAL, "%s: NULL pointer in the cache", who);
	if (((uintptr_t)c->table | (uintptr_t)c->len) & 3) return set_err(TG_CUDA_EINVAL, "%s: table or len is not on a 4-byte boundary", who);
	c->page_stride = pg_stride(c->page_stride, c->pages, e), c->head_stride = pg_stride(c->head_stride, c->nkv, e), c->pos_stride = pg_stride(c->pos_stride, c->page, e);
	if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15) || ((c->page_stride | c->head_stride | c->pos_stride) * e & 15))
		return set_err(TG_CUDA_EINVAL, "%s: cache rows must start on 16-byte boundaries", who);
	if (c->page_stride < 0 || c->head_stride < 0 || c->pos_stride < 0) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	o->shift = 4;
	while (o->shift < 30 && !(((c->page_stride | c->pos_stride) * e) >> o->shift & 1)) o->shift++;
	if (c->pages && ((unsigned __int128)c->page_stride * (c->pages - 1) + (unsigned __int128)c->pos_stride * (c->page - 1)) * e >> o->shift >= PG_NONE)
		return set_err(TG_CUDA_EINVAL, "%s: a pool of 2^32 rows' alignments of %d bytes or more", who, 1 << o->shift);
	o->k = (char *)c->k, o->v = (char *)c->v, o->table = c->table, o->len = c->len;
	o->page_b = c->page_stride * e, o->head_b = c->head_stride * e, o->pos_b = c->pos_stride * e;
	o->page = c->page, o->pages = c->pages, o->cols = c->table_cols, o->max_len = c->max_len;
	o->nkv = c->nkv, o->dim = c->head_dim;
	return TG_CUDA_OK;
}

int pg_drafts(const char *who, const tg_cuda_kv *c, const tg_cuda_drafts *desc, int use, int most, PgDrafts *o)
{
	if (!desc) return set_err(TG_CUDA_EINVAL, "%s: NULL drafted tokens", who);
	tg_cuda_drafts copy = *desc, *d = &copy;
	if (d->tokens <= 0 || (most && d->tokens > most)) return set_err(TG_CUDA_EINVAL, "%s: %d tokens per sequence", who, d->tokens);
	const int e = pg_size(c->type);
	d->q_seq = pg_stride(d->q_seq, c->seqs, e), d->q_tok = pg_stride(d->q_tok, d->tokens, e), d->q_head = pg_stride(d->q_head, d->nq, e);
	d->kv_seq = pg_stride(d->kv_seq, c->seqs, e), d->kv_tok = pg_stride(d->kv_tok, d->tokens, e), d->kv_head = pg_stride(d->kv_head, c->nkv, e);
	if (use & PG_USE_Q) {
		if (d->nq <= 0 || d->nq > 1 << 20 || d->nq % c->nkv)
			return set_err(TG_CUDA_EINVAL, "%s: nq %d is not a multiple of nkv %d, or over 2^20", who, d->nq, c->nkv);
		if (c->seqs && !d->q) return set_err(TG_CUDA_EINVAL, "%s: NULL q", who);
		if (((uintptr_t)d->q & 15) || ((d->q_seq | d->q_tok | d->q_head) * e & 15))
			return set_err(TG_CUDA_EINVAL, "%s: q rows must start on 16-byte boundaries", who);
	}
	if (c->seqs && (((use & PG_USE_K) && !d->k) || ((use & PG_USE_V) && !d->v)))
		return set_err(TG_CUDA_EINVAL, "%s: NULL drafted k or v", who);
	if (((use & PG_USE_K) && ((uintptr_t)d->k & 15)) || ((use & PG_USE_V) && ((uintptr_t)d->v & 15)) ||
	    ((d->kv_seq | d->kv_tok | d->kv_head) * e & 15))
		return set_err(TG_CUDA_EINVAL, "%s: drafted k and v rows must start on 16-byte boundaries", who);
	if (((use & PG_USE_Q) && (d->q_seq < 0 || d->q_tok < 0 || d->q_head < 0)) || d->kv_seq < 0 || d->kv_tok < 0 || d->kv_head < 0)
		return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	if (((uintptr_t)d->mask & 7) || ((uintptr_t)d->count & 3)) return set_err(TG_CUDA_EINVAL, "%s: mask (8 bytes) or count (4) is not on a boundary of its type", who);
	// attention passes on places within a sequence's drafted rows in 32 bits of 16 bytes
	if (most && (((unsigned __int128)d->kv_tok * d->tokens * e >> 4) >= PG_NONE ||
		     (((unsigned __int128)d->q_tok * d->tokens + (unsigned __int128)d->q_head * d->nq) * e >> 4) >= PG_NONE))
		return set_err(TG_CUDA_EINVAL, "%s: a sequence's drafted rows span 64 GB", who);
	o->q = (const char *)d->q, o->k = (const char *)d->k, o->v = (const char *)d->v;
	o->q_seq = d->q_seq * e, o->q_tok = d->q_tok * e, o->q_head = d->q_head * e;
	o->kv_seq = d->kv_seq * e, o->kv_tok = d->kv_tok * e, o->kv_head = d->kv_head * e;
	o->mask = d->mask, o->count = d->count, o->tokens = d->tokens, o->scale = d->scale;
	o->nq = use & PG_USE_Q ? d->nq : c->nkv, o->group = o->nq / c->nkv;
	return TG_CUDA_OK;
}

int pg_apart(const char *who, const char *what, int row, std::array<long long, 3> stride, std::array<int, 3> n)
{
	for (int i = 0; i < 2; i++) // ascending strides
		for (int k = 0; k < 2; k++)
			if (stride[k] > stride[k + 1]) std::swap(stride[k], stride[k + 1]), std::swap(n[k], n[k + 1]);
	__int128 span = row;
	for (int i = 0; i < 3; i++) {
		if (n[i] <= 1) continue;
		if (stride[i] < span) return set_err(TG_CUDA_EINVAL, "%s: rows of %s overlap (a stride of %lld)", who, what, stride[i]);
		span += (__int128)stride[i] * (n[i] - 1);
	}
	return TG_CUDA_OK;
}

// The dimensions of more than one row, ascending; a stride of 0 adds no rows.
struct PgDims {
	__int128 row;
	int count = 0;
	long long stride[3];
	long long n[3];

	explicit PgDims(const PgRows &x) : row(x.row)
	{
		for (int i = 0; i < 3; i++) {
			if (x.n[i] <= 1 || x.stride[i] == 0) continue;
			int k = count++;
			for (; k && stride[k - 1] > x.stride[i]; k--) stride[k] = stride[k - 1], n[k] = n[k - 1];
			stride[k] = x.stride[i], n[k] = x.n[i];
		}
	}
	__int128 span(int dims) const // of its first dimensions
	{
		__int128 s = row;
		for (int i = 0; i < dims; i++) s += (__int128)stride[i] * (n[i] - 1);
		return s;
	}
};

// b's rows `off` bytes behind a's, of the first na and nb dimensions
static bool dims_meet(const PgDims &a, int na, const PgDims &b, int nb, __int128 off)
{
	if (off >= a.span(na) || off + b.span(nb) <= 0) return false;
	if (!na && !nb) return true;
	const long long s = std::max(na ? a.stride[na - 1] : 0, nb ? b.stride[nb - 1] : 0);
	const int ia = na && a.stride[na - 1] == s ? na - 1 : na, ib = nb && b.stride[nb - 1] == s ? nb - 1 : nb; // what lies within a step of s
	if (a.span(ia) > s || b.span(ib) > s) return true;
	const __int128 ca = ia < na ? a.n[ia] : 1, cb = ib < nb ? b.n[ib] : 1;
	const __int128 j = -(off >= 0 ? off / s : -((-off + s - 1) / s)); // b's element x + j begins less than s behind a's element x, x + j - 1 before it
	for (__int128 k = j - 1; k <= j; k++)
		if (k > -ca && k < cb && dims_meet(a, ia, b, ib, off + k * s)) return true;
	return false;
}

bool pg_meet(const PgRows &a, const PgRows &b)
{
	for (const PgRows *x : { &a, &b })
		if (!x->at || x->row <= 0 || x->n[0] <= 0 || x->n[1] <= 0 || x->n[2] <= 0) return false;
	const __int128 off = (__int128)(uintptr_t)b.at - (__int128)(uintptr_t)a.at;
	auto span = [](const PgRows &x) {
		__int128 n = x.row;
		for (int i = 0; i < 3; i++) n += (__int128)x.stride[i] * (x.n[i] - 1);
		return n;
	};
	if (off >= span(a) || off + span(b) <= 0) return false; // nearly always
	const PgDims da(a), db(b);
	return dims_meet(da, da.count, db, db.count, off);
}

int pg_len_out(const char *who, const tg_cuda_kv *c, const tg_cuda_drafts *d, const int *len_out)
{
	auto ints = [&](const int *at) -> PgRows { return { at, 4ll * c->seqs, {}, { 1, 1, 1 } }; };
	if (pg_meet(ints(len_out), ints(c->len))) return set_err(TG_CUDA_EINVAL, "%s: len_out may not share memory with the cache's len", who);
	if (pg_meet(ints(len_out), ints(d->count))) return set_err(TG_CUDA_EINVAL, "%s: len_out may not share memory with count", who);
	return TG_CUDA_OK;
}

bool pg_map(CUtensorMap *m, const PgCache &c, const void *pool, bool f16, int rows, PgBox *box)
{
	static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
	static std::once_flag once;
	std::call_once(once, [] {
		cudaDriverEntryPointQueryResult q;
		void *fn = nullptr;
		if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
			encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
	});
	box->rows = std::min(rows, c.page), box->swap = c.head_b < c.pos_b;
	const long long first = std::min(c.head_b, c.pos_b), second = std::max(c.head_b, c.pos_b);
	if (!encode || c.pages <= 0 || c.page % 8 || (rows % c.page && c.page % rows) || first <= 0 || second % first || c.page_b % second || c.page_b <= 0 ||
	    c.page_b >= 1ll << 40)
		return false;
	const cuuint64_t dims[4] = { (cuuint64_t)c.dim, (cuuint64_t)(box->swap ? c.nkv : c.page), (cuuint64_t)(box->swap ? c.page : c.nkv), (cuuint64_t)c.pages };
	const cuuint64_t strides[3] = { (cuuint64_t)first, (cuuint64_t)second, (cuuint64_t)c.page_b };
	const cuuint32_t size[4] = { 64, (cuuint32_t)(box->swap ? 1 : box->rows), (cuuint32_t)(box->swap ? box->rows : 1), 1 }, es[4] = { 1, 1, 1, 1 };
	return encode(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void *)pool, dims, strides, size, es,
		      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
		      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---- commit -------------------------------------------------------------------------------

struct CommitArgs {
	PgCache c;
	PgDrafts d;
	const int *path;
	int *len_out;
	const float *fresh;
	float *acc;
	long long acc_seq, acc_head;
	int acc_cols, seqs, chunks, lg; // chunks: 16-byte pieces of a row; lg: their logarithm where they are a power of two, else -1
};

// A copy, bound by HBM: one warp per (sequence, accepted token); its lanes take the 16-byte
// pieces of all heads' rows, so a drafted token's rows (contiguous in the usual layout)
// are read and written in whole sectors. Measured: 32 prompts of 1024 tokens (8 heads of 128, f32) 90 us,
// 6.0 TB/s (101 us with one piece at a time).
__global__ void __launch_bounds__(256) k_commit(const CommitArgs p)
{
	const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
	const int lane = threadIdx.x & 31;
	const long long b = w / p.d.tokens;
	const int i = (int)(w - b * p.d.tokens);
	if (b >= p.seqs) return;
	const int n = p.c.length((int)b), cnt = p.d.drafted((int)b);
	if (i == 0 && lane == 0) p.len_out[b] = p.c.grown(n, cnt);
	if (i >= cnt) return;
	const int from = p.path ? p.path[b * p.d.tokens + i] : i;
	const long long at = (long long)n + i;
	if ((unsigned)from >= (unsigned)p.d.tokens) {
		p.c.report(PG_PATH);
		return;
	}
	if (at >= (long long)p.c.page * p.c.cols || at > 0x7fffffff) {
		p.c.report(PG_ROOM);
		return;
	}
	const long long to = p.c.row(p.c.table + b * p.c.cols, (int)at);
	if (to < 0) return;
	const long long src = b * p.d.kv_seq + from * p.d.kv_tok;
	const int all = p.c.nkv * p.chunks;
	for (int x0 = 0; x0 < all; x0 += 4 * 32) { // four pieces of K and of V a lane on their way at once
		uint4 k[4], v[4];
		long long to4[4];
#pragma unroll
		for (int u = 0; u < 4; u++) {
			const int x = x0 + u * 32 + lane, h = p.lg >= 0 ? x >> p.lg : x / p.chunks, o = (x - h * p.chunks) * 16;
			to4[u] = x < all ? to + h * p.c.head_b + o : -1;
			if (x < all) {
				k[u] = __ldcs((const uint4 *)(p.d.k + src + h * p.d.kv_head + o));
				v[u] = __ldcs((const uint4 *)(p.d.v + src + h * p.d.kv_head + o));
			}
		}
#pragma unroll
		for (int u = 0; u < 4; u++)
			if (to4[u] >= 0) *(uint4 *)(p.c.k + to4[u]) = k[u], *(uint4 *)(p.c.v + to4[u]) = v[u];
	}
	if (!p.acc) return;
	if (at >= p.acc_cols) {
		if (lane == 0) p.c.report(PG_ROOM);
		return;
	}
	for (int h = lane; h < p.c.nkv; h += 32)
		p.acc[b * p.acc_seq + h * p.acc_head + at] = p.fresh[(b * p.c.nkv + h) * p.d.tokens + from];
}

} // namespace tgc

using namespace tgc;

extern "C" int tg_cuda_kv_commit(const tg_cuda_kv *c, const tg_cuda_drafts *d, const int *path, int *len_out, const float *fresh,
				 float *acc, long long acc_seq, long long acc_head, int acc_cols, void *stream)
{
	const char *who = "tg_cuda_kv_commit";
	clear_err();
	CommitArgs p = {};
	int rc, sms;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_K | PG_USE_V, 0, &p.d))) return rc;
	if (c->seqs && (!len_out || !fresh != !acc)) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (((uintptr_t)path | (uintptr_t)len_out | (uintptr_t)fresh | (uintptr_t)acc) & 3) return set_err(TG_CUDA_EINVAL, "%s: a pointer is not on a 4-byte boundary", who);
	if ((rc = pg_len_out(who, c, d, len_out))) return rc;
	if (acc && acc_cols < 0) return set_err(TG_CUDA_EINVAL, "%s: acc_cols %d", who, acc_cols);
	if (acc && (rc = pg_apart(who, "acc", acc_cols, {acc_seq, acc_head, 0}, {c->seqs, c->nkv, 1}))) return rc;
	if ((rc = pg_apart(who, "the cache", c->head_dim, {c->page_stride, c->head_stride, c->pos_stride}, {c->pages, c->nkv, c->page}))) return rc;
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0) return rc;
	p.path = path, p.len_out = len_out, p.fresh = fresh, p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head;
	p.acc_cols = acc_cols, p.seqs = c->seqs, p.chunks = c->head_dim * pg_size(c->type) / 16;
	p.lg = -1;
	if (!(p.chunks & (p.chunks - 1)))
		for (p.lg = 0; 1 << p.lg < p.chunks;) p.lg++;
	const long long blocks = ((long long)c->seqs * d->tokens + 7) / 8;
	if (blocks > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of %d tokens", who, c->seqs, d->tokens);
	k_commit<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}
