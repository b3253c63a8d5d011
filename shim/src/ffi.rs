// Generated by shim/gen_ffi.py from include/zkb200.h, zkb200_air.h and zkb200_prover.h. Do not edit by hand.
// One declaration per exported function of libzkb200.so; status codes as in zkb200.h (0 = ok, < 0 = error).
#![allow(non_snake_case, clippy::too_many_arguments)]

#[repr(C)] pub struct ZkbCtx { _private: [u8; 0] }  // zkb_ctx: opaque
#[repr(C)] pub struct ZkbAirProgram { _private: [u8; 0] }  // zkb_air_program: opaque
#[repr(C)] pub struct ZkbShardPcs { _private: [u8; 0] }  // zkb_shard_pcs: opaque

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbGrid {
    pub log_rows: u32,
    pub groups: u32,
    pub chunks: u32,
    pub lead: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbDequantCfg {
    pub variant: u32,
    pub sticky: u32,
    pub kmax: u32,
    pub do_ref: u32,
    pub tokens: u32,
    pub n_out: u32,
    pub per_row: u32,
    pub chunks: u32,
    pub log_rows: u32,
    pub slot0: u32,
    pub per_slot: u32,
    pub chan_w: u32,
    pub f_acc: u32,
    pub f_sg: u32,
    pub f_m2: u32,
    pub f_ph: u32,
    pub f_st: u32,
    pub f_r: u32,
    pub f_m7: u32,
    pub f_ef: u32,
    pub f_nz: u32,
    pub f_eo: u32,
    pub f_mul: [u32; 6],
    pub sh0: u32,
    pub sh1: u32,
    pub n_norm: u32,
    pub n_frac: u32,
    pub n_mul: u32,
    pub n_r8: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbRsGroup {
    pub n: u32,
    pub leaf_col: u32,
    pub width: u32,
    pub un: u32,
    pub flat: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbRsSlot {
    pub a_sm: u32,
    pub a_ef: u32,
    pub b_sm: u32,
    pub b_ef: u32,
    pub base: u32,
    pub o_sm: u32,
    pub o_ef: u32,
    pub from_slot: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbRsProgram {
    pub groups: *const ZkbRsGroup,
    pub n_groups: u32,
    pub slots: *const ZkbRsSlot,
    pub n_slots: u32,
    pub out_slot: *const u32,
    pub out_w: u32,
    pub kind: u32,
    pub sticky: u32,
    pub kmax: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbRsTables {
    pub norm3: *const u32,
    pub n_norm: u32,
    pub smul3: *const i32,
    pub n_smul: u32,
    pub const un2: *mut *const i32,
    pub n_un: u32,
    pub n_val: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbRsMult {
    pub m: *mut u32,
    pub n: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbRsMults {
    pub pow: ZkbRsMult,
    pub norm: ZkbRsMult,
    pub val: ZkbRsMult,
    pub frac: ZkbRsMult,
    pub smul: ZkbRsMult,
    pub un: *const ZkbRsMult,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbStepEmbedArgs {
    pub ids: *const i32,
    pub table: *const std::ffi::c_void,
    pub row_scale: *const f32,
    pub out: *mut std::ffi::c_void,
    pub off_table: *mut u64,
    pub table_stride: i64,
    pub out_stride: i64,
    pub segment_stride: i64,
    pub n_tokens: u32,
    pub vocab: u32,
    pub width: u32,
    pub segment: u32,
    pub table_type: u32,
    pub out_type: u32,
    pub scale: f32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbKvCache {
    pub k: *mut std::ffi::c_void,
    pub v: *mut std::ffi::c_void,
    pub k_scale: *mut f32,
    pub v_scale: *mut f32,
    pub seq_stride: i64,
    pub head_stride: i64,
    pub token_stride: i64,
    pub scale_seq_stride: i64,
    pub scale_head_stride: i64,
    pub ty: u32,
    pub n_seqs: u32,
    pub n_heads: u32,
    pub head_dim: u32,
    pub capacity: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbStepRows {
    pub first: *const i32,
    pub kv_len: *const i32,
    pub n_rows: u32,
    pub max_rows: u32,
    pub max_len: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbStepNormRopeArgs {
    pub cache: ZkbKvCache,
    pub rows: ZkbStepRows,
    pub q: *const std::ffi::c_void,
    pub k: *const std::ffi::c_void,
    pub v: *const std::ffi::c_void,
    pub q_weight: *const u16,
    pub k_weight: *const u16,
    pub h_inv_freq: *const f64,
    pub q_out: *mut std::ffi::c_void,
    pub q_stride: i64,
    pub k_stride: i64,
    pub v_stride: i64,
    pub head_stride: i64,
    pub q_out_stride: i64,
    pub q_out_head_stride: i64,
    pub ty: u32,
    pub q_heads: u32,
    pub rotary_dim: u32,
    pub interleaved: u32,
    pub eps: f32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbStepAttentionArgs {
    pub cache: ZkbKvCache,
    pub rows: ZkbStepRows,
    pub q: *const std::ffi::c_void,
    pub out: *mut std::ffi::c_void,
    pub q_stride: i64,
    pub q_head_stride: i64,
    pub out_stride: i64,
    pub out_head_stride: i64,
    pub q_heads: u32,
    pub out_type: u32,
    pub window: u32,
    pub sinks: u32,
    pub scale: f32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbAirOp {
    pub op: u32,
    pub a: u32,
    pub b: u32,
    pub c: u32,
    pub d: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbAirStats {
    pub n_ops: u32,
    pub n_live_ops: u32,
    pub n_uniform: u32,
    pub n_instr: u32,
    pub n_loads: u32,
    pub n_columns_read: u32,
    pub reg_words: u32,
    pub uniform_words: u32,
    pub threads: u32,
    pub rows_per_thread: u32,
    pub smem_bytes: u32,
    pub m31_mults: u32,
    pub specialized: u32,
    pub specialized_regs: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug, Default)]
pub struct ZkbPcsConfig {
    pub pow_bits: u32,
    pub log_blowup_factor: u32,
    pub log_last_layer_degree_bound: u32,
    pub n_queries: u32,
}

#[repr(C)] #[derive(Copy, Clone, Debug)]
pub struct ZkbStarkComponent {
    pub prog: *mut ZkbAirProgram,
    pub trace_log: u32,
    pub scalars: *const u32,
    pub claimed_sum: *const u32,
}

extern "C" {
    pub fn zkb_init(device: i32, max_log_size: i32, out: *mut *mut ZkbCtx) -> i32;
    pub fn zkb_destroy(ctx: *mut ZkbCtx) -> i32;
    pub fn zkb_last_error(ctx: *mut ZkbCtx) -> *const std::os::raw::c_char;
    pub fn zkb_sync(ctx: *mut ZkbCtx) -> i32;
    pub fn zkb_get_stream(ctx: *mut ZkbCtx, stream: *mut *mut std::ffi::c_void) -> i32;
    pub fn zkb_max_log_size(ctx: *mut ZkbCtx) -> i32;
    pub fn zkb_event_record(ctx: *mut ZkbCtx, slot: i32) -> i32;
    pub fn zkb_event_elapsed_ms(ctx: *mut ZkbCtx, a: i32, b: i32, h_ms: *mut f32) -> i32;
    pub fn zkb_profile_begin(ctx: *mut ZkbCtx) -> i32;
    pub fn zkb_profile_end(ctx: *mut ZkbCtx, h_names: *mut *const std::os::raw::c_char, h_ms: *mut f32, h_count: *mut i32, cap: i32, n: *mut i32) -> i32;
    pub fn zkb_fft_arith_ceiling(ctx: *mut ZkbCtx, h_butterflies_per_s: *mut f64) -> i32;
    pub fn zkb_malloc(ctx: *mut ZkbCtx, bytes: usize, dptr: *mut *mut std::ffi::c_void) -> i32;
    pub fn zkb_free(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void) -> i32;
    pub fn zkb_memset_zero(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_h2d(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void, h_src: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_d2h(ctx: *mut ZkbCtx, h_dst: *mut std::ffi::c_void, dptr: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_h2d_async(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void, h_pinned_src: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_d2h_async(ctx: *mut ZkbCtx, h_pinned_dst: *mut std::ffi::c_void, dptr: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_h2d_overlapped(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void, h_pinned_src: *const std::ffi::c_void, bytes: usize, fence: i32) -> i32;
    pub fn zkb_wait_fence(ctx: *mut ZkbCtx, fence: i32) -> i32;
    pub fn zkb_peer_buffer_alloc(ctx: *mut ZkbCtx, bytes: usize, dptr: *mut *mut std::ffi::c_void, handle: *mut u8) -> i32;
    pub fn zkb_peer_buffer_free(ctx: *mut ZkbCtx, dptr: *mut std::ffi::c_void) -> i32;
    pub fn zkb_peer_buffer_open(ctx: *mut ZkbCtx, handle: *const u8, peer_ptr: *mut *mut std::ffi::c_void) -> i32;
    pub fn zkb_peer_buffer_close(ctx: *mut ZkbCtx, peer_ptr: *mut std::ffi::c_void) -> i32;
    pub fn zkb_copy_to_peer(ctx: *mut ZkbCtx, dst: *mut std::ffi::c_void, src: *const std::ffi::c_void, bytes: usize, lane: i32) -> i32;
    pub fn zkb_peer_copies_wait(ctx: *mut ZkbCtx) -> i32;
    pub fn zkb_d2d(ctx: *mut ZkbCtx, dst: *mut std::ffi::c_void, src: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn zkb_host_alloc_pinned(ctx: *mut ZkbCtx, bytes: usize, h_ptr: *mut *mut std::ffi::c_void) -> i32;
    pub fn zkb_host_free_pinned(ctx: *mut ZkbCtx, h_ptr: *mut std::ffi::c_void) -> i32;
    pub fn zkb_gather_multi(ctx: *mut ZkbCtx, cols: *const *const u32, ncols: i32, h_idx: *const u32, nidx: i32, h_out: *mut u32) -> i32;
    pub fn zkb_gather_hashes(ctx: *mut ZkbCtx, hashes: *const u32, h_idx: *const u32, nidx: i32, h_out: *mut u32) -> i32;
    pub fn zkb_gather_words(ctx: *mut ZkbCtx, h_addrs: *const *const u32, n: usize, h_out: *mut u32) -> i32;
    pub fn zkb_twiddles_d2h(ctx: *mut ZkbCtx, log_size: i32, h_tw: *mut u32, h_itw: *mut u32) -> i32;
    pub fn zkb_ifft_cols(ctx: *mut ZkbCtx, cols: *const *mut u32, ncols: i32, log_n: i32) -> i32;
    pub fn zkb_lde_cols(ctx: *mut ZkbCtx, coeffs: *const *const u32, ncols: i32, log_n: i32, out: *const *mut u32, log_out: i32) -> i32;
    pub fn zkb_eval_at_point_cols(ctx: *mut ZkbCtx, coeffs: *const *const u32, ncols: i32, log_n: i32, h_point: *const u32, h_out: *mut u32) -> i32;
    pub fn zkb_barycentric_weights(ctx: *mut ZkbCtx, log_size: i32, h_point: *const u32, d_weights: *mut u32) -> i32;
    pub fn zkb_barycentric_eval_at_point(ctx: *mut ZkbCtx, d_evals: *const u32, d_weights: *const u32, log_size: i32, h_out: *mut u32) -> i32;
    pub fn zkb_eval_at_point_by_folding(ctx: *mut ZkbCtx, d_evals: *const u32, log_size: i32, h_point: *const u32, h_out: *mut u32) -> i32;
    pub fn zkb_fri_decompose(ctx: *mut ZkbCtx, d_eval: *const *const u32, log_size: i32, d_out: *const *mut u32, h_lambda: *mut u32) -> i32;
    pub fn zkb_bit_reverse_m31(ctx: *mut ZkbCtx, col: *mut u32, log_n: i32) -> i32;
    pub fn zkb_bit_reverse_qm31(ctx: *mut ZkbCtx, col: *mut u32, log_n: i32) -> i32;
    pub fn zkb_merkle_layer(ctx: *mut ZkbCtx, log_size: i32, prev: *const u32, cols: *const *const u32, ncols: i32, m31_out: i32, out: *mut u32) -> i32;
    pub fn zkb_merkle_leaves_partial(ctx: *mut ZkbCtx, log_size: i32, cols: *const *const u32, ncols: i32, cols_before: i32, total_cols: i32, m31_out: i32, out: *mut u32) -> i32;
    pub fn zkb_merkle_levels(ctx: *mut ZkbCtx, child_log: i32, children: *const u32, levels: i32, out_layers: *const *mut u32, m31_out: i32) -> i32;
    pub fn zkb_merkle_top(ctx: *mut ZkbCtx, top_log: i32, top_layer: *const u32, lower_layers: *const *mut u32, m31_out: i32) -> i32;
    pub fn zkb_merkle_top_channel(ctx: *mut ZkbCtx, top_log: i32, top_layer: *const u32, lower_layers: *const *mut u32, m31_out: i32, d_chan: *mut u32, d_alpha: *mut u32, d_root_copy: *mut u32) -> i32;
    pub fn zkb_fold_circle_into_line(ctx: *mut ZkbCtx, dst: *const *mut u32, src: *const *const u32, log_n_src: i32, h_alpha: *const u32) -> i32;
    pub fn zkb_fold_line_dalpha(ctx: *mut ZkbCtx, out: *const *mut u32, inp: *const *const u32, log_n: i32, d_alpha: *const u32) -> i32;
    pub fn zkb_fold_circle_into_line_dalpha(ctx: *mut ZkbCtx, dst: *const *mut u32, src: *const *const u32, log_n_src: i32, d_alpha: *const u32) -> i32;
    pub fn zkb_channel_mix_root_draw(ctx: *mut ZkbCtx, d_chan: *mut u32, d_root: *const u32, d_alpha: *mut u32, d_root_copy: *mut u32) -> i32;
    pub fn zkb_fold_line_dalpha_leaves(ctx: *mut ZkbCtx, out: *const *mut u32, inp: *const *const u32, log_n: i32, d_alpha: *const u32, leaves: *mut u32) -> i32;
    pub fn zkb_fold_circle_into_line_dalpha_leaves(ctx: *mut ZkbCtx, dst: *const *mut u32, src: *const *const u32, log_n_src: i32, d_alpha: *const u32, leaves: *mut u32) -> i32;
    pub fn zkb_fold_line(ctx: *mut ZkbCtx, out: *const *mut u32, inp: *const *const u32, log_n: i32, h_alpha: *const u32) -> i32;
    pub fn zkb_quot_numerators(ctx: *mut ZkbCtx, cols: *const *const u32, ncols: i32, log_n: i32, h_col_idx: *const u32, h_b: *const u32, h_c: *const u32, k: i32, out: *const *mut u32) -> i32;
    pub fn zkb_quot_combine(ctx: *mut ZkbCtx, n_acc: i32, acc_cols: *const *const u32, h_acc_log: *const i32, h_first_lin: *const u32, h_points: *const u32, lifting_log: i32, out: *const *mut u32) -> i32;
    pub fn zkb_quot_combine_rows(ctx: *mut ZkbCtx, n_acc: i32, acc_cols: *const *const u32, h_acc_log: *const i32, h_first_lin: *const u32, h_points: *const u32, lifting_log: i32, row_begin: usize, n_rows: usize, out: *const *mut u32) -> i32;
    pub fn zkb_accumulate(ctx: *mut ZkbCtx, col: *const *mut u32, other: *const *const u32, n: usize) -> i32;
    pub fn zkb_lift_accumulate(ctx: *mut ZkbCtx, dst: *const *mut u32, log_dst: i32, src: *const *const u32, log_src: i32) -> i32;
    pub fn zkb_secure_powers(ctx: *mut ZkbCtx, h_felt: *const u32, n: usize, h_out: *mut u32) -> i32;
    pub fn zkb_gkr_eq_evals(ctx: *mut ZkbCtx, h_y: *const u32, ny: i32, h_v: *const u32, out: *mut u32) -> i32;
    pub fn zkb_gkr_next_layer(ctx: *mut ZkbCtx, kind: i32, num: *const u32, den: *const u32, n: usize, num_out: *mut u32, den_out: *mut u32) -> i32;
    pub fn zkb_gkr_sum(ctx: *mut ZkbCtx, kind: i32, num: *const u32, den: *const u32, n: usize, eq_evals: *const u32, h_lambda: *const u32, h_out: *mut u32) -> i32;
    pub fn zkb_gkr_fix_and_sum(ctx: *mut ZkbCtx, kind: i32, num: *const u32, den: *const u32, n: usize, h_r: *const u32, eq_evals: *const u32, h_lambda: *const u32, num_out: *mut u32, den_out: *mut u32, h_out: *mut u32) -> i32;
    pub fn zkb_mle_fix_qm31(ctx: *mut ZkbCtx, inp: *const u32, n: usize, h_r: *const u32, out: *mut u32) -> i32;
    pub fn zkb_mle_fix_m31(ctx: *mut ZkbCtx, inp: *const u32, n: usize, h_r: *const u32, out: *mut u32) -> i32;
    pub fn zkb_gkr_sum_noalloc(device: i32, stream: *mut std::ffi::c_void, kind: i32, num: *const u32, den: *const u32, n: usize, eq_evals: *const u32, h_lambda: *const u32, d_out: *mut u32) -> i32;
    pub fn zkb_gkr_sum_noalloc_error() -> *const std::os::raw::c_char;
    pub fn zkb_grind(ctx: *mut ZkbCtx, h_prefixed_digest: *const u32, pow_bits: i32, m31_out: i32, h_nonce: *mut u64) -> i32;
    pub fn zkb_freivalds_scatter(ctx: *mut ZkbCtx, qx: *const i8, qw: *const *const i8, h_n_out: *const u32, grid: *const ZkbGrid, pq: u32, pk: u32, n_in: u32, tokens: u32, n_mats: u32, base_cols: *const *mut u32, pre_cols: *const *mut u32, m_r8: *mut u32, table_len: u32, off_table: *mut u64) -> i32;
    pub fn zkb_freivalds_acc(ctx: *mut ZkbCtx, base_cols: *const *const u32, pre_cols: *const *const u32, grid: *const ZkbGrid, pq: u32, pk: u32, n_mats: u32, h_s: *const u32, h_rv: *const u32, out_cols: *const *mut u32, h_claims: *mut u32) -> i32;
    pub fn zkb_witness_tables(ctx: *mut ZkbCtx, expmap: *const u32, counters: *const *const u32, n_counters: u32, patch_idx: *const u32, patch_val: *const u32, n_patch: u32, log_rows: u32, bf16x: i32, two_pow: f64, x_col: *mut u32, y_col: *mut u32, m_col: *mut u32) -> i32;
    pub fn zkb_witness_dequant(ctx: *mut ZkbCtx, acc: *const i32, jx: *const i32, jw: *const i32, sx: *const u32, sw: *const u32, norm3: *const u32, mul2: *const u32, base_cols: *const *mut u32, n_base: u32, pre_cols: *const *mut u32, n_pre: u32, m_norm: *mut u32, m_frac: *mut u32, m_mul: *mut u32, m_r8: *mut u32, counts: *mut u32, want_out: *mut u32, cfg: *const ZkbDequantCfg) -> i32;
    pub fn zkb_witness_pre_table(ctx: *mut ZkbCtx, kind: u32, log_rows: u32, kmax: u32, round: u32, counters: *const *const u32, n_counters: u32, patch_idx: *const u32, patch_val: *const u32, n_patch: u32, cols: *const *mut u32, n_cols: u32, m_col: *mut u32) -> i32;
    pub fn zkb_key_tile_flags(ctx: *mut ZkbCtx, shape: u32, log_rows: u32, groups: u32, chunks: u32, lead: u32, descending: u32, modulus: u32, rw: u32, flags: *mut u32) -> i32;
    pub fn zkb_witness_selectors(ctx: *mut ZkbCtx, shape: u32, log_rows: u32, groups: u32, chunks: u32, lead: u32, descending: u32, flags: *const u32, scale: *const u32, ctx_len: u32, n_insts: u32, with_scale: i32, cols: *const *mut u32, n_cols: u32) -> i32;
    pub fn zkb_witness_residual_stream(ctx: *mut ZkbCtx, prog: *const ZkbRsProgram, tables: *const ZkbRsTables, wit: *const u32, live_rows: u32, log_rows: u32, cols: *const *mut u32, n_cols: u32, out_pat: *mut u32, out_nat: *mut i32, in_nat: *mut i32, mults: *const ZkbRsMults, counts: *mut u32) -> i32;
    pub fn zkb_step_embed(ctx: *mut ZkbCtx, args: *const ZkbStepEmbedArgs) -> i32;
    pub fn zkb_step_norm_rope(ctx: *mut ZkbCtx, args: *const ZkbStepNormRopeArgs) -> i32;
    pub fn zkb_step_attention(ctx: *mut ZkbCtx, args: *const ZkbStepAttentionArgs) -> i32;
    pub fn zkb_air_compile(ctx: *mut ZkbCtx, ops: *const ZkbAirOp, n_ops: usize, constraints: *const u32, n_constraints: usize, tree_cols: *const u32, n_trees: i32, n_scalars: usize, out: *mut *mut ZkbAirProgram) -> i32;
    pub fn zkb_air_free(prog: *mut ZkbAirProgram) -> i32;
    pub fn zkb_air_specialize(ctx: *mut ZkbCtx, prog: *mut ZkbAirProgram) -> i32;
    pub fn zkb_air_select(prog: *mut ZkbAirProgram, specialized: i32) -> i32;
    pub fn zkb_air_get_stats(prog: *const ZkbAirProgram, out: *mut ZkbAirStats) -> i32;
    pub fn zkb_air_analyze(ops: *const ZkbAirOp, n_ops: usize, constraints: *const u32, n_constraints: usize, tree_cols: *const u32, n_trees: i32, n_scalars: usize, check_specialized: i32, out: *mut ZkbAirStats, err: *mut std::os::raw::c_char, err_cap: usize) -> i32;
    pub fn zkb_constraint_quotients(ctx: *mut ZkbCtx, prog: *const ZkbAirProgram, cols: *const *const u32, scalars: *const u32, cumsum_shift: *const u32, random_coeff_powers: *const u32, denom_inv: *const u32, trace_log: i32, eval_log: i32, accum: *const *mut u32, accumulate: i32) -> i32;
    pub fn zkb_constraint_denom_inv(trace_log: i32, eval_log: i32, out: *mut u32) -> i32;
    pub fn zkb_pcs_prove_device(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, d_cols: *const *mut u32, col_logs: *const u32, config: *const ZkbPcsConfig, two_sample_every: i32, h_out: *mut u32, cap: usize, n_words: *mut usize, h_phase_ms: *mut f32) -> i32;
    pub fn zkb_pcs_prove_host(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, h_cols: *const *const u32, col_logs: *const u32, config: *const ZkbPcsConfig, two_sample_every: i32, h_out: *mut u32, cap: usize, n_words: *mut usize, h_phase_ms: *mut f32) -> i32;
    pub fn zkb_stark_prove_device(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, d_cols: *const *mut u32, trace_log: u32, prog: *mut ZkbAirProgram, scalars: *const u32, claimed_sum: *const u32, config: *const ZkbPcsConfig, h_out: *mut u32, cap: usize, n_words: *mut usize, oods_evals: *mut u32, h_phase_ms: *mut f32, composition_ms: *mut f32) -> i32;
    pub fn zkb_stark_prove_host(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, h_cols: *const *const u32, trace_log: u32, prog: *mut ZkbAirProgram, scalars: *const u32, claimed_sum: *const u32, config: *const ZkbPcsConfig, h_out: *mut u32, cap: usize, n_words: *mut usize, oods_evals: *mut u32, h_phase_ms: *mut f32, composition_ms: *mut f32) -> i32;
    pub fn zkb_stark_prove_multi_device(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, d_cols: *const *mut u32, n_components: i32, components: *const ZkbStarkComponent, config: *const ZkbPcsConfig, h_out: *mut u32, cap: usize, n_words: *mut usize, oods_evals: *mut u32, h_phase_ms: *mut f32, composition_ms: *mut f32) -> i32;
    pub fn zkb_stark_prove_multi_host(ctx: *mut ZkbCtx, n_trees: i32, tree_ncols: *const i32, h_cols: *const *const u32, n_components: i32, components: *const ZkbStarkComponent, config: *const ZkbPcsConfig, h_out: *mut u32, cap: usize, n_words: *mut usize, oods_evals: *mut u32, h_phase_ms: *mut f32, composition_ms: *mut f32) -> i32;
    pub fn zkb_gkr_prove_device(ctx: *mut ZkbCtx, n_inst: i32, kinds: *const i32, d_nums: *const *const u32, d_dens: *const *const u32, ns: *const u64, seed: u64, h_out: *mut u32, cap: usize, n_words: *mut usize) -> i32;
    pub fn zkb_shard_pcs_begin(ctx: *mut ZkbCtx, rank: i32, world: i32, ncols_total: i32, log_n: i32, config: *const ZkbPcsConfig, out: *mut *mut ZkbShardPcs) -> i32;
    pub fn zkb_shard_pcs_extend(s: *mut ZkbShardPcs, d_cols: *const *mut u32, d_send: *mut *mut u32, d_rows: *mut *mut u32) -> i32;
    pub fn zkb_shard_pcs_set_rows(s: *mut ZkbShardPcs, d_rows: *mut u32) -> i32;
    pub fn zkb_shard_pcs_set_peer_rows(s: *mut ZkbShardPcs, peer_rows: *const *mut u32) -> i32;
    pub fn zkb_shard_pcs_extend_begin(s: *mut ZkbShardPcs, d_cols: *const *mut u32, n_chunks: i32) -> i32;
    pub fn zkb_shard_pcs_extend_chunk(s: *mut ZkbShardPcs, k: i32, d_send: *mut *mut u32, d_recv: *mut *mut u32, words_per_peer: *mut usize) -> i32;
    pub fn zkb_shard_pcs_subtree(s: *mut ZkbShardPcs, d_root: *mut *mut u32, d_roots: *mut *mut u32) -> i32;
    pub fn zkb_shard_pcs_sample(s: *mut ZkbShardPcs, h_samples: *mut u32) -> i32;
    pub fn zkb_shard_pcs_quotients(s: *mut ZkbShardPcs, h_all_samples: *const u32, d_quot_local: *mut *mut u32, d_quot_full: *mut *mut u32) -> i32;
    pub fn zkb_shard_pcs_fri_and_decommit(s: *mut ZkbShardPcs, h_part: *mut u32, cap: usize, n_words: *mut usize) -> i32;
    pub fn zkb_shard_pcs_finish(s: *mut ZkbShardPcs, h_parts: *const *const u32, part_words: *const usize, h_out: *mut u32, cap: usize, n_words: *mut usize) -> i32;
    pub fn zkb_shard_pcs_end(s: *mut ZkbShardPcs) -> i32;
}
