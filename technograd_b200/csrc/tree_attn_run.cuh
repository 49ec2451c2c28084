// tree_attn_run.cuh -- the launches of a planned attention call, instantiated per element type.
#pragma once

#include "tree_attn.cuh"
#include "tree_attn_fma.cuh"
#include "tree_attn_tc.cuh"

namespace tgc {

// Units shared by many CTAs (few units) have many parts each: eight warps a block for them.
template <class T, int DP, int RT>
static int attn_join(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	if (pl.grid >= 4ll * pl.units) TGC_CUDA(launch_pdl(k_attn_join<T, DP, RT, 8>, dim3(pl.by_unit ? pl.units : pl.grid, RT * DP / 256), dim3(256), 0, st, p));
	else TGC_CUDA(launch_pdl(k_attn_join<T, DP, RT, 1>, dim3(pl.by_unit ? pl.units : pl.grid, RT * DP / 256), dim3(32), 0, st, p));
	return TG_CUDA_OK;
}

template <class T, int DP, int MT>
static int attn_run(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	using A = AttnTile<T, DP, MT>;
	static std::atomic<unsigned long long> done{0};
	int rc = pg_smem(k_tree_attn<T, DP, MT>, A::SMEM, pl.dev, done);
	if (rc) return rc;
	if (pl.whole) { // one kernel: the plain launch is the cheaper one for the host
		k_tree_attn<T, DP, MT><<<pl.grid, 128, A::SMEM, st>>>(p);
		TGC_LAUNCH_CHECK();
		return TG_CUDA_OK;
	}
	TGC_CUDA(launch_pdl(k_tree_attn<T, DP, MT>, dim3(pl.grid), dim3(128), A::SMEM, st, p));
	return attn_join<T, DP, A::RT>(p, pl, st);
}

template <int DP, int R>
static int attn_run_fma(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	using A = FmaTile<DP, R>;
	static std::atomic<unsigned long long> done{0};
	int rc = pg_smem(k_tree_attn_fma<DP, R>, A::SMEM, pl.dev, done);
	if (rc) return rc;
	if (pl.whole) {
		k_tree_attn_fma<DP, R><<<pl.grid, 128, A::SMEM, st>>>(p);
		TGC_LAUNCH_CHECK();
		return TG_CUDA_OK;
	}
	TGC_CUDA(launch_pdl(k_tree_attn_fma<DP, R>, dim3(pl.grid), dim3(128), A::SMEM, st, p));
	return attn_join<float, DP, R>(p, pl, st);
}

template <class T, int DP, bool BOX>
static int attn_run_tc(const AttnArgs &p, const AttnPlan &pl, const CUtensorMap *maps, cudaStream_t st)
{
	using A = TaTile<DP>;
	static std::atomic<unsigned long long> done{0};
	auto *kernel = k_tree_attn_tc<T, DP, BOX>;
	if (!(done.load(std::memory_order_acquire) >> pl.dev & 1)) { // the roles' registers must be the launch's: a warp would wait for ever for others
		cudaFuncAttributes at;
		TGC_CUDA(cudaFuncGetAttributes(&at, kernel));
		if (at.numRegs < TA_REGS) return set_err(TG_CUDA_EUNSUPPORTED, "tree attention kernel built with %d registers, not %d", at.numRegs, TA_REGS);
	}
	int rc = pg_smem(kernel, A::SMEM, pl.dev, done);
	if (rc) return rc;
	TGC_CUDA(launch_pdl(kernel, dim3(pl.grid), dim3(A::THREADS), A::SMEM, st, p, maps[0], maps[1]));
	return pl.whole ? TG_CUDA_OK : attn_join<T, DP, A::RT>(p, pl, st);
}

// Pages that suit boxes have a kernel of their own: one kernel with both ways of fetching costs the other pages (24 rows, trees of
// 21 tokens over 8 sequences of up to 1280 positions) 29.4 us where 26.8 do, and copies cost pages of 64 (48 sequences of up
// to 6001 positions, 64 tokens) 257 us where boxes take 248, pages of 16 (131009 positions, 40 rows) 88 us against 84.
template <class T, int DP>
static int attn_run_tc(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	AttnArgs a = p;
	CUtensorMap maps[2] = {};
	const bool f16 = std::is_same<T, __half>::value;
	if (pg_map(&maps[0], p.c, p.c.k, f16, 64, &a.box) && pg_map(&maps[1], p.c, p.c.v, f16, 64, &a.box)) return attn_run_tc<T, DP, true>(a, pl, maps, st);
	return attn_run_tc<T, DP, false>(a, pl, maps, st);
}

template <class T>
int attn_type(const AttnArgs &p, const AttnPlan &pl, cudaStream_t st)
{
	if constexpr (sizeof(T) == 2) {
		if (pl.tc) return pl.dp == 128 ? attn_run_tc<T, 128>(p, pl, st) : attn_run_tc<T, 64>(p, pl, st);
	}
	if constexpr (sizeof(T) == 4) {
		if (pl.fma == 4) return pl.dp == 256 ? attn_run_fma<256, 4>(p, pl, st) : pl.dp == 128 ? attn_run_fma<128, 4>(p, pl, st) : attn_run_fma<64, 4>(p, pl, st);
		if (pl.fma == 8) return pl.dp == 256 ? attn_run_fma<256, 8>(p, pl, st) : pl.dp == 128 ? attn_run_fma<128, 8>(p, pl, st) : attn_run_fma<64, 8>(p, pl, st);
	}
	if (pl.dp == 256) return attn_run<T, 256, 1>(p, pl, st);
	if (pl.dp == 128) return pl.mt == 1 ? attn_run<T, 128, 1>(p, pl, st) : attn_run<T, 128, 2>(p, pl, st);
	return pl.mt == 1 ? attn_run<T, 64, 1>(p, pl, st) : attn_run<T, 64, 2>(p, pl, st);
}

} // namespace tgc
