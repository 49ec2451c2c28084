// attn_weights.cu -- tg_cuda_attn_weights: the attention weight that a paged cache's positions receive.
#include "common.cuh"
#include "mma_sync.cuh"
#include "paged.cuh"

namespace tgc {

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

// One CTA per (sequence, kv head, chunk of 64 KB of keys), the drafted tokens a chunk of their own after
// the cached ones. A warp keeps its keys in shared memory and meets the query rows 32 at a time, as
// k_tree_attn does: S = Q K^T, then the sum over rows of 2^(z - lse log2(e)) for each key stays in
// registers until the last rows. Bound by HBM while the rows are few: keys are read once, three CTAs
// per SM keep their loads in flight; by the tensor cores from about 64 rows on.
template <class T, int DP> struct WeightTile {
	static constexpr int KW = sizeof(T) == 4 ? 8 : 16, NT = KW / 8, MT = 2, RB = 32;
	static constexpr int P = DP * (int)sizeof(T), CH = P / 16;
	static constexpr int KC = 65536 / P, NG = KC / 4 / KW; // keys per CTA; groups of KW keys per warp
	static constexpr int K = RB * P, LSE = K + KC * P, MASK = LSE + RB * 4, SMEM = MASK + RB * 8;
};

template <class T, int DP>
__global__ void __launch_bounds__(128) k_attn_weights(const WeightArgs p)
{
	using W = WeightTile<T, DP>;
	constexpr int KW = W::KW, NT = W::NT, MT = W::MT, RB = W::RB, P = W::P, CH = W::CH, NG = W::NG, MINE = NG * KW;
	extern __shared__ __align__(128) char smem[];
	float *s_lse = (float *)(smem + W::LSE);
	unsigned long long *s_mask = (unsigned long long *)(smem + W::MASK);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
	const uint32_t s0 = smem_u32(smem), sk = s0 + W::K + warp * MINE * P;
	pdl_launch();
	pdl_wait();
	long long r = blockIdx.x;
	const int chunk = (int)(r % p.chunks);
	r /= p.chunks;
	const int h = (int)(r % p.c.nkv), b = (int)(r / p.c.nkv);
	const int n = p.c.length(b), cnt = p.d.drafted(b), chunks = p.c.dim * (int)sizeof(T) / 16;
	const unsigned long long sel = p.select ? p.select[b] : ~0ull;
	const bool drafted = chunk == p.chunks - 1;
	const long long x0 = (drafted ? 0 : (long long)chunk * W::KC) + warp * MINE; // this warp's first key
	const int end = drafted ? cnt : n;
	const float zs = p.d.scale * 1.4426950408889634f;
	float acc[NG][NT][2];
#pragma unroll
	for (int i = 0; i < NG; i++)
#pragma unroll
		for (int x = 0; x < NT; x++) acc[i][x][0] = acc[i][x][1] = 0;
	const bool any = (drafted ? 0 : (long long)chunk * W::KC) < end; // of the CTA
	const int groups = x0 < end ? (int)min((long long)NG, (end - x0 + KW - 1) / KW) : 0;
	if (any) {
		for (int i = 0; i < groups; i++) {
			const char *kp = nullptr;
			const long long x = x0 + i * KW + lane;
			if (lane < KW && x < end) {
				if (drafted) kp = p.d.k + (long long)b * p.d.kv_seq + x * p.d.kv_tok + h * p.d.kv_head;
				else {
					const long long at = p.c.row(p.c.table + (long long)b * p.c.cols, (int)x);
					if (at >= 0) kp = p.c.k + at + h * p.c.head_b;
				}
			}
#pragma unroll
			for (int y = 0; y < KW * CH / 32; y++) {
				const int z = y * 32 + lane, row = z / CH, ch = z % CH;
				const unsigned long long kr = __shfl_sync(~0u, (unsigned long long)kp, row);
				const bool have = kr && ch < chunks;
				cp16(sk + (i * KW + row) * P + ((ch ^ (row & 7)) << 4), have ? (const char *)kr + ch * 16 : p.d.k, have);
			}
		}
		cp_commit();
		const int rows = p.d.tokens * p.d.group;
		for (int r0 = 0; r0 < rows; r0 += RB) {
			__syncthreads();
			for (int x = tid; x < RB * CH; x += 128) {
				const int row = x / CH, ch = x % CH, rr = r0 + row, t = rr / p.d.group;
				uint4 v = make_uint4(0, 0, 0, 0);
				if (rr < rows && ch < chunks)
					v = *(const uint4 *)(p.d.q + (long long)b * p.d.q_seq + (long long)t * p.d.q_tok + (long long)(h * p.d.group + rr % p.d.group) * p.d.q_head + ch * 16);
				*(uint4 *)(smem + row * P + ((ch ^ (row & 7)) << 4)) = v;
			}
			if (tid < RB) { // the row's lse, and which drafted keys it counts for (cached ones: all or none)
				const int rr = r0 + tid, t = rr / p.d.group;
				const bool in = rr < rows && t < cnt && (sel >> t & 1);
				const float lse = in ? p.lse[((long long)b * p.d.tokens + t) * p.d.nq + h * p.d.group + rr % p.d.group] : -INFINITY;
				s_lse[tid] = lse * 1.4426950408889634f;
				s_mask[tid] = lse == -INFINITY ? 0 : drafted ? p.d.sees(b, t, cnt) : ~0ull;
			}
			cp_wait<0>();
			__syncthreads();
#pragma unroll
			for (int i = 0; i < NG; i++) {
				if (i >= groups) break;
				float s[MT][NT][4];
#pragma unroll
				for (int m = 0; m < MT; m++)
#pragma unroll
					for (int x = 0; x < NT; x++) s[m][x][0] = s[m][x][1] = s[m][x][2] = s[m][x][3] = 0;
				qk_tile<T, DP, MT, NT>(s, s0, sk + i * KW * P, lane);
#pragma unroll
				for (int m = 0; m < MT; m++)
#pragma unroll
					for (int e = 0; e < 2; e++) {
						const int row = m * 16 + e * 8 + g;
						const float ref = s_lse[row];
						const unsigned long long ok = s_mask[row];
#pragma unroll
						for (int x = 0; x < NT; x++)
#pragma unroll
							for (int y = 0; y < 2; y++) {
								const bool in = drafted ? ok >> (warp * MINE + i * KW + x * 8 + 2 * t4 + y) & 1 : ok != 0;
								acc[i][x][y] += in ? ex2(s[m][x][2 * e + y] * zs - ref) : 0;
							}
					}
			}
		}
	}
	const long long head = (long long)b * p.c.nkv + h;
#pragma unroll
	for (int i = 0; i < NG; i++)
#pragma unroll
		for (int x = 0; x < NT; x++)
#pragma unroll
			for (int y = 0; y < 2; y++) {
				float w = acc[i][x][y]; // over the rows g, g + 8, ...: lanes of one t4
				w += __shfl_xor_sync(~0u, w, 4);
				w += __shfl_xor_sync(~0u, w, 8);
				w += __shfl_xor_sync(~0u, w, 16);
				const long long key = x0 + i * KW + x * 8 + 2 * t4 + y;
				if (g) continue;
				if (drafted) {
					if (key < p.d.tokens) p.fresh[head * p.d.tokens + key] = key < end ? w : 0;
				} else if (key < p.c.max_len)
					p.acc_out[head * p.c.max_len + key] = key < end ? (p.acc ? p.acc[b * p.acc_seq + h * p.acc_head + key] : 0) + w : 0;
			}
}

template <class T, int DP>
static int weights_run(WeightArgs &p, int seqs, int dev, cudaStream_t st, const char *who)
{
	using W = WeightTile<T, DP>;
	static std::atomic<unsigned long long> done{0};
	int rc = pg_smem(k_attn_weights<T, DP>, W::SMEM, dev, done);
	if (rc) return rc;
	p.chunks = (p.c.max_len + W::KC - 1) / W::KC + 1;
	const long long blocks = (long long)seqs * p.c.nkv * p.chunks;
	if (blocks > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences of up to %d positions", who, seqs, p.c.max_len);
	TGC_CUDA(launch_pdl(k_attn_weights<T, DP>, dim3((unsigned)blocks), dim3(128), W::SMEM, st, p));
	return TG_CUDA_OK;
}

template <class T>
static int weights_type(WeightArgs &p, int seqs, int dev, cudaStream_t st, const char *who)
{
	if (p.c.dim > 128) return weights_run<T, 256>(p, seqs, dev, st, who);
	return p.c.dim > 64 ? weights_run<T, 128>(p, seqs, dev, st, who) : weights_run<T, 64>(p, seqs, dev, st, who);
}

} // namespace tgc

using namespace tgc;

extern "C" int tg_cuda_attn_weights(const tg_cuda_kv *c, const tg_cuda_drafts *d, const float *lse, const unsigned long long *select,
				    const float *acc, long long acc_seq, long long acc_head, float *acc_out, float *fresh, void *stream)
{
	const char *who = "tg_cuda_attn_weights";
	clear_err();
	WeightArgs p = {};
	int rc, sms, dev;
	if ((rc = pg_cache(who, c, &p.c)) || (rc = pg_drafts(who, c, d, PG_USE_Q | PG_USE_K, 64, &p.d))) return rc;
	if (c->seqs && (!lse || !fresh || (!acc_out && c->max_len))) return set_err(TG_CUDA_EINVAL, "%s: NULL pointer", who);
	if (acc && acc == acc_out && (acc_head != c->max_len || acc_seq != (long long)c->nkv * c->max_len))
		return set_err(TG_CUDA_EINVAL, "%s: acc may be acc_out with acc_out's own strides only", who);
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0 || (rc = pg_sms(who, &dev, &sms))) return rc;
	p.lse = lse, p.select = select, p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head, p.acc_out = acc_out, p.fresh = fresh;
	cudaStream_t st = (cudaStream_t)stream;
	return c->type == TG_CUDA_F32 ? weights_type<float>(p, c->seqs, dev, st, who)
	       : c->type == TG_CUDA_F16 ? weights_type<__half>(p, c->seqs, dev, st, who)
					: weights_type<__nv_bfloat16>(p, c->seqs, dev, st, who);
}
