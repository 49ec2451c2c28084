// attn_weights.cu -- tg_cuda_attn_weights: the attention weight that a paged cache's positions receive.
#include <type_traits>

#include "attn_weights_tc.cuh"

namespace tgc {

// The weights' kernel goes through the keys as k_tree_attn does (tree_attn.cuh): equal shares of all
// (sequence, kv head) units' tiles, a ring of asynchronous copies per warp, drafted tokens after the cached
// ones. A warp takes its tile's keys into registers as the product's operand and meets all query rows
// with them, 16 at a time from shared memory: S = Q K^T, then exp(scale s - lse) summed over the rows in
// registers and, at the tile's end, over lanes. Every key is one warp's, so nothing is joined and results
// do not depend on timing. Up to QR rows stay in shared memory for a unit; more are taken in turns at
// every tile.
// What bounds it: latency where the shares are short, then instruction issue (about 540 a warp for 16 keys and 64 rows);
// 16-bit caches with long shares take attn_weights_tc.cuh (rule and figures below). Measured: one token of 16 query heads over 8
// sequences of up to 1280 positions 14.4 us a call.
template <class T, int DP> struct WeightTile {
	// eight warps where the keys' registers allow two such CTAs per SM: the products' latencies need them
	static constexpr int NW = sizeof(T) == 2 && DP <= 128 ? 8 : 4, THREADS = 32 * NW;
	static constexpr int KW = sizeof(T) == 4 ? 8 : 16, NT = KW / 8, TK = NW * KW;
	static constexpr int P = DP * (int)sizeof(T), CH = P / 16, STAGE = KW * P, NST = NW == 8 || DP == 256 ? 2 : 4;
	static constexpr int QR = 32768 / P; // 32 KB of rows
	static constexpr int RING = QR * P, LSE = RING + NW * NST * STAGE, MASK = LSE + QR * 4, SCAN = MASK + QR * 8, SMEM = SCAN + (NW + 4) * 8;
};

template <class T, int DP>
__global__ void __launch_bounds__(WeightTile<T, DP>::THREADS, 2) k_attn_weights(const WeightArgs p)
{
	using W = WeightTile<T, DP>;
	constexpr int KW = W::KW, NT = W::NT, TK = W::TK, P = W::P, CH = W::CH, NST = W::NST, QR = W::QR, THREADS = W::THREADS;
	extern __shared__ __align__(128) char smem[];
	float *s_lse = (float *)(smem + W::LSE);
	unsigned long long *s_mask = (unsigned long long *)(smem + W::MASK);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
	const uint32_t s0 = smem_u32(smem), ring = s0 + W::RING + warp * NST * W::STAGE;
	const int extra = (p.d.tokens + TK - 1) / TK, rows = p.d.tokens * p.d.group, chunks = p.c.dim * (int)sizeof(T) / 16;
	const int turns = (rows + QR - 1) / QR;
	AttnCursor c;
	long long left, pos, share;
	if (!attn_share<TK, W::NW>(p, (long long *)(smem + W::SCAN), extra, c, left, pos, share)) return;

	// ---- fetching: lane i < KW holds the place of the tile's key i, looked up while the tile before is fetched
	AttnCursor f = c;
	long long fetched = 0;
	uint32_t at = PG_NONE;
	auto find = [&]() {
		at = PG_NONE;
		if (lane >= KW || fetched >= left) return;
		if (f.tile < f.ctx) {
			const int x = f.tile * TK + warp * KW + lane;
			if (x < f.n) {
				const int page = x / p.c.page;
				at = p.c.at(p.c.table[(long long)f.b * p.c.cols + page], x - page * p.c.page);
			}
		} else {
			const int u = (f.tile - f.ctx) * TK + warp * KW + lane;
			if (u < p.d.drafted(f.b)) at = (uint32_t)(u * p.d.kv_tok >> 4);
		}
	};
	auto fetch = [&](int stage) {
		if (fetched < left) {
			const bool ctx = f.tile < f.ctx;
			const int sh = ctx ? p.c.shift : 4;
			const char *kp = (ctx ? p.c.k : p.d.k) + (ctx ? f.h * p.c.head_b : f.b * p.d.kv_seq + f.h * p.d.kv_head);
			const uint32_t sk = ring + stage * W::STAGE, mine = at;
			cursor_next<TK>(p, f, extra);
			fetched++;
			find();
#pragma unroll
			for (int i = 0; i < KW * CH / 32; i++) {
				const int row = (i * 32 + lane) / CH, ch = (i * 32 + lane) % CH;
				const uint32_t r = __shfl_sync(~0u, mine, row);
				const bool have = r != PG_NONE && ch < chunks;
				cp16(sk + row * P + ((ch ^ (row & 7)) << 4), have ? kp + ((unsigned long long)r << sh) + ch * 16 : p.d.k, have);
			}
		}
		cp_commit();
	};
	find();
#pragma unroll
	for (int i = 0; i < NST - 1; i++) fetch(i);

	// rows r0 .. r0 + QR of unit c into shared memory: q, lse, and the drafted tokens each counts for
	// (cached positions: all bits or none)
	auto load_rows = [&](int r0) {
		const int cnt = p.d.drafted(c.b), in = min(QR, (rows - r0 + 15) & ~15);
		const unsigned long long sel = p.select ? p.select[c.b] : ~0ull;
		for (int x = tid; x < in * CH; x += THREADS) {
			const int row = x / CH, ch = x % CH, r = r0 + row, t = r / p.d.group;
			const bool have = r < rows && ch < chunks;
			cp16(s0 + row * P + ((ch ^ (row & 7)) << 4),
			     have ? p.d.q + (long long)c.b * p.d.q_seq + (long long)t * p.d.q_tok + (long long)(c.h * p.d.group + r - t * p.d.group) * p.d.q_head + ch * 16 : p.d.k, have);
		}
		for (int x = tid; x < in; x += THREADS) {
			const int r = r0 + x, t = r / p.d.group;
			const bool on = r < rows && t < cnt && (sel >> t & 1);
			const float lse = on ? p.lse[((long long)c.b * p.d.tokens + t) * p.d.nq + c.h * p.d.group + r - t * p.d.group] : -INFINITY;
			s_lse[x] = lse;
			s_mask[x] = lse == -INFINITY ? 0 : p.d.sees(c.b, t, cnt);
		}
		cp_commit();
		cp_wait<0>();
	};

	int stage = 0;
	bool first = true;
	for (long long i = 0; i < left; i++) {
		if (first && turns == 1) { // a unit begins here, or goes on from the CTA before
			__syncthreads();
			load_rows(0);
			__syncthreads();
		}
		fetch((stage + NST - 1) % NST);
		cp_wait<NST - 1>();
		__syncwarp();
		const bool drafted = c.tile >= c.ctx;
		const int x0 = (drafted ? c.tile - c.ctx : c.tile) * TK + warp * KW, end = drafted ? p.d.drafted(c.b) : c.n; // this warp's first key
		const long long head = (long long)c.b * p.c.nkv + c.h;
		// what the keys had: lane (g = 0, t4) has keys x0 + 8 x + 2 t4 and the next
		float had[NT][2], acc[NT][2];
#pragma unroll
		for (int x = 0; x < NT; x++)
#pragma unroll
			for (int y = 0; y < 2; y++) {
				const int key = x0 + x * 8 + 2 * t4 + y;
				had[x][y] = g == 0 && !drafted && p.acc && key < end ? p.acc[c.b * p.acc_seq + c.h * p.acc_head + key] : 0;
				acc[x][y] = 0;
			}
		KeyFrag<T, DP> k;
		load_keys<T, DP>(k, ring + stage * W::STAGE, lane);
		for (int turn = 0; turn < turns; turn++) {
			if (turns > 1) {
				__syncthreads();
				load_rows(turn * QR);
				__syncthreads();
			}
			const int tiles = (min(QR, rows - turn * QR) + 15) / 16;
			auto meet = [&](auto mt, int m0) { // mt tiles of 16 rows at once, from m0 on
				constexpr int MT = decltype(mt)::value;
				float s[MT][NT][4];
				qk_keys<T, DP, MT, NT>(s, k, s0 + m0 * 16 * P, lane);
				unsplit_scores<T, DP, MT, NT>(s, s0 + m0 * 16 * P, ring + stage * W::STAGE, lane);
#pragma unroll
				for (int m = 0; m < MT; m++)
#pragma unroll
					for (int e = 0; e < 2; e++) {
						const int row = (m0 + m) * 16 + e * 8 + g;
						const float ref = s_lse[row];
						if (drafted) {
							const unsigned long long ok = x0 < 64 ? s_mask[row] >> (x0 + 2 * t4) : 0; // (a mask's bits end at 64, a tile may not)
#pragma unroll
							for (int x = 0; x < NT; x++)
#pragma unroll
								for (int y = 0; y < 2; y++) acc[x][y] += ok >> (x * 8 + y) & 1 ? weight_of(s[m][x][2 * e + y], p.d.scale, ref) : 0;
						} else {
#pragma unroll
							for (int x = 0; x < NT; x++)
#pragma unroll
								for (int y = 0; y < 2; y++) acc[x][y] += ref != -INFINITY ? weight_of(s[m][x][2 * e + y], p.d.scale, ref) : 0;
						}
					}
			};
			int m = 0;
			for (; m + 4 <= tiles; m += 4) meet(std::integral_constant<int, 4>(), m);
			if (tiles - m >= 2) meet(std::integral_constant<int, 2>(), m), m += 2;
			if (tiles > m) meet(std::integral_constant<int, 1>(), m);
		}
#pragma unroll
		for (int x = 0; x < NT; x++)
#pragma unroll
			for (int y = 0; y < 2; y++) {
				float w = acc[x][y]; // over the rows g, g + 8, ...: lanes of one t4
				w += __shfl_xor_sync(~0u, w, 4);
				w += __shfl_xor_sync(~0u, w, 8);
				w += __shfl_xor_sync(~0u, w, 16);
				const int key = x0 + x * 8 + 2 * t4 + y;
				if (g) continue;
				if (drafted) {
					if (key < p.d.tokens) p.fresh[head * p.d.tokens + key] = key < end ? w : 0;
				} else if (key < end) p.acc_out[head * p.c.max_len + key] = had[x][y] + w;
			}
		if (c.tile == c.ctx) // the cached positions' end: nothing is past it
			for (long long x = (long long)c.n + tid; x < p.c.max_len; x += THREADS) p.acc_out[head * p.c.max_len + x] = 0;
		first = c.tile == c.all - 1;
		__syncwarp(); // every lane is done with this stage
		stage = (stage + 1) % NST;
		cursor_next<TK>(p, c, extra);
	}
	cp_wait<0>();
}

template <class T, int DP>
static int weights_run(WeightArgs &p, int sms, int dev, cudaStream_t st, const char *who)
{
	using W = WeightTile<T, DP>;
	static std::atomic<unsigned long long> done{0};
	int rc = pg_smem(k_attn_weights<T, DP>, W::SMEM, dev, done);
	if (rc) return rc;
	const long long units = (long long)p.seqs * p.c.nkv, tiles = (p.c.max_len + W::TK - 1) / W::TK + (p.d.tokens + W::TK - 1) / W::TK;
	if (units > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences", who, p.seqs);
	p.row_tiles = 1, p.whole = 0, p.least = W::TK < 128 ? 128 / W::TK : 1, p.begin = 1, p.split = nullptr;
	const long long shares = (units * (tiles + p.begin) + p.least + p.begin - 1) / (p.least + p.begin), wave = 2ll * sms;
	k_attn_weights<T, DP><<<(unsigned)(shares < wave ? shares : wave), W::THREADS, W::SMEM, st>>>(p);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

template <class T, int DP>
static int weights_run_tc(WeightArgs &p, int sms, int dev, cudaStream_t st, const char *who)
{
	using W = TwTile<DP>;
	static std::atomic<unsigned long long> done{0};
	int rc = pg_smem(k_attn_weights_tc<T, DP>, W::SMEM, dev, done);
	if (rc) return rc;
	const long long units = (long long)p.seqs * p.c.nkv, tiles = (p.c.max_len + W::TK - 1) / W::TK + 1;
	if (units > 0x7fffffff) return set_err(TG_CUDA_EINVAL, "%s: %d sequences", who, p.seqs);
	// a unit's start is worth about 4 tiles (32-token windows, us at 2, 4, 6 and 8: 16 sequences of up to 16001 positions 131, 91, 89,
	// 91; 16 of up to 6001 61, 48, 50, 52; 32 of up to 1280 37.6, 34, 35.6, 37.6; 8 of up to 1280 21, 20, 20.7, 21)
	p.row_tiles = 1, p.whole = 0, p.least = 1, p.begin = 4, p.split = nullptr;
	const long long shares = (units * (tiles + p.begin) + p.begin) / (1 + p.begin);
	CUtensorMap map = {};
	if (!pg_map(&map, p.c, p.c.k, std::is_same<T, __half>::value, 32, &p.box)) p.box.rows = 0;
	k_attn_weights_tc<T, DP><<<(unsigned)(shares < sms ? shares : sms), W::THREADS, W::SMEM, st>>>(p, map);
	TGC_LAUNCH_CHECK();
	return TG_CUDA_OK;
}

// Of up to TW_ROWS query rows per key head, 16-bit caches take attn_weights_tc.cuh where a CTA has more than so many of its tiles,
// whatever the rows: below, latency decides, and this file's kernel has more CTAs and warps. Measured, us, tiles of 128 keys
// against this file's (8 key heads, bf16, 2 / 32 / 64 / 256 rows), at 128 dimensions 17.9, 18.5, 23.3, 59 and 17, 19.1, 23.7, 68 at
// 10 tiles a CTA; 21.4, 21.9, 29.3, 81 and 25.2, 29.4, 35.4, 114 at 16; 27.2, 27.2, 36.1, 103 and 32.3, 37.5, 48.5, 161 at 29;
// 69, 70, 92, 271 and 106, 121, 150, 538 at 110. At 64 dimensions 20.8, 21, 27.2, 71 and 20.5, 23.1, 27.8, 58 at 16; 25.1, 25.2, 33.5, 92
// and 25.2, 29.3, 35.6, 76 at 29; 33.4, 33.5, 43.7, 124 and 37.6, 45.7, 55.5, 118 at 42; 62, 63, 85, 231 and 90, 102, 121, 246 at 110.
constexpr int WEIGHTS_TC_TILES_128 = 14, WEIGHTS_TC_TILES_64 = 40;

template <class T>
static int weights_type(WeightArgs &p, int sms, int dev, cudaStream_t st, const char *who)
{
	if constexpr (sizeof(T) == 2) {
		const long long tiles = (long long)p.seqs * p.c.nkv * ((p.c.max_len + 127) / 128 + 1);
		if (p.c.dim <= 128 && p.d.tokens * p.d.group <= TW_ROWS && tiles > (long long)(p.c.dim > 64 ? WEIGHTS_TC_TILES_128 : WEIGHTS_TC_TILES_64) * sms)
			return p.c.dim > 64 ? weights_run_tc<T, 128>(p, sms, dev, st, who) : weights_run_tc<T, 64>(p, sms, dev, st, who);
	}
	if (p.c.dim > 128) return weights_run<T, 256>(p, sms, dev, st, who);
	return p.c.dim > 64 ? weights_run<T, 128>(p, sms, dev, st, who) : weights_run<T, 64>(p, sms, dev, st, who);
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
	if (((uintptr_t)select & 7) || (((uintptr_t)lse | (uintptr_t)acc | (uintptr_t)acc_out | (uintptr_t)fresh) & 3))
		return set_err(TG_CUDA_EINVAL, "%s: a pointer is not on a boundary of its type", who);
	if (acc && ((acc_seq < 0 && c->seqs > 1) || (acc_head < 0 && c->nkv > 1))) return set_err(TG_CUDA_EINVAL, "%s: negative strides", who);
	if (acc && acc == acc_out && (acc_head != c->max_len || acc_seq != (long long)c->nkv * c->max_len))
		return set_err(TG_CUDA_EINVAL, "%s: acc may be acc_out with acc_out's own strides only", who);
	if ((rc = pg_device(who, &sms, &p.c.status)) || c->seqs == 0 || (rc = pg_sms(who, &dev, &sms))) return rc;
	p.seqs = c->seqs, p.lse = (float *)lse, p.select = select, p.acc = acc, p.acc_seq = acc_seq, p.acc_head = acc_head, p.acc_out = acc_out, p.fresh = fresh;
	cudaStream_t st = (cudaStream_t)stream;
	return c->type == TG_CUDA_F32 ? weights_type<float>(p, sms, dev, st, who)
	       : c->type == TG_CUDA_F16 ? weights_type<__half>(p, sms, dev, st, who)
					: weights_type<__nv_bfloat16>(p, sms, dev, st, who);
}
