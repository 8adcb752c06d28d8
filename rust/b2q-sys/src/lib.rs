// Generated by gen_ffi.py from include/b2q.h: do not edit by hand.
//! Raw bindings of libb2q.so, the sm_100a quantized linear-layer kernels behind a C ABI.
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_int, c_void};

#[repr(C)] pub struct b2q_handle_s { _private: [u8; 0] }
pub type b2q_handle = *mut b2q_handle_s;
#[repr(C)] pub struct b2q_tp_s { _private: [u8; 0] }
pub type b2q_tp = *mut b2q_tp_s;

#[repr(C)] #[derive(Debug, Clone, Copy, Default, PartialEq, Eq)]
pub struct b2q_tile_config { pub tile_m: u32, pub tile_n: u32, pub tile_k: u32, pub warp_m: u32, pub warp_n: u32, pub stages: u32, pub use_tensor_core: u32, pub split_k: u32 }
#[repr(C)] #[derive(Debug, Clone, Copy)]
pub struct b2q_gemm_fp8_problem { pub a: *const u8, pub w: *const u8, pub m: i64, pub n: i64, pub k: i64, pub scale_a: *const f32, pub scale_a_kind: i32, pub scale_w: *const f32, pub scale_w_kind: i32, pub out: *mut c_void }
#[repr(C)] #[derive(Debug, Clone, Copy)]
pub struct b2q_gemm_fp8_desc { pub a: *const u8, pub w: *const u8, pub m: i64, pub n: i64, pub k: i64, pub fmt: i32, pub scale_a: *const f32, pub scale_a_kind: i32, pub scale_w: *const f32, pub scale_w_kind: i32, pub out: *mut c_void, pub out_type: i32, pub alpha: f32, pub beta: f32, pub bias: *const f32, pub epilogue: i32, pub w_layout: i32 }

pub const B2Q_OK: i32 = 0;
pub const B2Q_ERR_CUDA: i32 = 1;
pub const B2Q_ERR_INVALID_DIMENSION: i32 = 2;
pub const B2Q_ERR_BUFFER_TOO_SMALL: i32 = 3;
pub const B2Q_ERR_DIMENSION_MISMATCH: i32 = 4;
pub const B2Q_ERR_UNSUPPORTED: i32 = 5;
pub const B2Q_ERR_LAUNCH_FAILED: i32 = 7;
pub const B2Q_ERR_INVALID_ARGUMENT: i32 = 8;
pub const B2Q_ERR_EMPTY_INPUT: i32 = 20;
pub const B2Q_ERR_GROUP_SIZE_MISMATCH: i32 = 21;
pub const B2Q_ERR_INVALID_SCALE: i32 = 22;
pub const B2Q_ERR_NON_FINITE_FP8: i32 = 23;
pub const B2Q_ERR_INVALID_CONFIG: i32 = 24;
pub const B2Q_ERR_INVALID_BIT_WIDTH: i32 = 25;
pub const B2Q_ERR_TIMEOUT: i32 = 40;
pub const B2Q_ERR_NCCL: i32 = 41;
pub const B2Q_FP8_E4M3: i32 = 0;
pub const B2Q_FP8_E5M2: i32 = 1;
pub const B2Q_ROUND_REF: i32 = 0;
pub const B2Q_ROUND_RNE: i32 = 1;
pub const B2Q_FP4_E2M1: i32 = 0;
pub const B2Q_FP4_INT4: i32 = 1;
pub const B2Q_SCALE_F32: i32 = 0;
pub const B2Q_SCALE_E8M0: i32 = 1;
pub const B2Q_SYMMETRIC: i32 = 0;
pub const B2Q_ASYMMETRIC: i32 = 1;
pub const B2Q_OUT_BF16: i32 = 0;
pub const B2Q_OUT_F32: i32 = 1;
pub const B2Q_SCALE_SCALAR: i32 = 0;
pub const B2Q_SCALE_PER_ROW: i32 = 1;
pub const B2Q_KV_PER_TOKEN: i32 = 0;
pub const B2Q_KV_PER_CHANNEL: i32 = 1;
pub const B2Q_EPI_LINEAR: i32 = 0;
pub const B2Q_EPI_RELU: i32 = 1;
pub const B2Q_EPI_GELU: i32 = 2;
pub const B2Q_EPI_BIAS: i32 = 3;
pub const B2Q_EPI_BIAS_RELU: i32 = 4;
pub const B2Q_EPI_SWIGLU: i32 = 5;
pub const B2Q_W_NK: i32 = 0;
pub const B2Q_W_KN: i32 = 1;
pub const B2Q_GATE_UP_CONCATENATED: i32 = 0;
pub const B2Q_GATE_UP_INTERLEAVED128: i32 = 1;
pub const B2Q_FP4_ACT_SPLIT: i32 = 0;
pub const B2Q_FP4_ACT_MXFP8: i32 = 1;
pub const B2Q_GGML_Q8_0: i32 = 0;
pub const B2Q_GGML_Q4_0: i32 = 1;
pub const B2Q_GGML_Q4_1: i32 = 2;
pub const B2Q_GGML_Q4_K: i32 = 3;

#[link(name = "b2q")]
extern "C" {
    pub fn b2q_create(out: *mut b2q_handle, device: c_int) -> i32;
    pub fn b2q_destroy(h: b2q_handle) -> i32;
    pub fn b2q_set_stream(h: b2q_handle, stream: *mut c_void) -> i32;
    pub fn b2q_set_static_weights(h: b2q_handle, static_weights: c_int) -> i32;
    pub fn b2q_get_sm(h: b2q_handle, sm: *mut c_int) -> i32;
    pub fn b2q_get_sm_count(h: b2q_handle, count: *mut c_int) -> i32;
    pub fn b2q_last_error(h: b2q_handle) -> *const c_char;
    pub fn b2q_check(h: b2q_handle) -> i32;
    pub fn b2q_minmax_calibrate_f32(h: b2q_handle, x: *const f32, rows: i64, cols: i64, bits: c_int, scheme: c_int, scales: *mut f32, zero_points: *mut i32) -> i32;
    pub fn b2q_minmax_quantize_f32(h: b2q_handle, x: *const f32, rows: i64, cols: i64, scales: *const f32, zero_points: *const i32, bits: c_int, scheme: c_int, codes: *mut i32) -> i32;
    pub fn b2q_minmax_dequantize_f32(h: b2q_handle, codes: *const i32, rows: i64, cols: i64, scales: *const f32, zero_points: *const i32, out: *mut f32) -> i32;
    pub fn b2q_fake_quant_inplace_f32(h: b2q_handle, x: *mut f32, n: i64, scale: f32, zero_point: f32, qmin: f32, qmax: f32) -> i32;
    pub fn b2q_fp8_encode_f32(h: b2q_handle, x: *const f32, n: i64, fmt: c_int, rounding: c_int, codes: *mut u8) -> i32;
    pub fn b2q_fp8_decode_f32(h: b2q_handle, codes: *const u8, n: i64, fmt: c_int, rounding: c_int, out: *mut f32) -> i32;
    pub fn b2q_fp8_remap_ref_subnormals(h: b2q_handle, codes: *mut u8, n: i64, fmt: c_int) -> i32;
    pub fn b2q_fp8_quantize_rows_f32(h: b2q_handle, x: *const f32, rows: i64, cols: i64, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8) -> i32;
    pub fn b2q_fp8_quantize_rows_bf16(h: b2q_handle, x_bf16: *const c_void, rows: i64, cols: i64, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8) -> i32;
    pub fn b2q_swiglu_quantize_rows_bf16(h: b2q_handle, gate: *const c_void, up: *const c_void, rows: i64, cols: i64, ld: i64, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8) -> i32;
    pub fn b2q_fp8_quantize_rows_f32_noalloc(x: *const f32, rows: i64, cols: i64, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8, stream: *mut c_void, device_status: *mut i32, err: *mut c_char, err_len: usize) -> i32;
    pub fn b2q_fp4_block_quantize_f32(h: b2q_handle, x: *const f32, n: i64, block: c_int, format: c_int, scale_format: c_int, packed: *mut u8, scales: *mut c_void) -> i32;
    pub fn b2q_fp4_block_dequantize_f32(h: b2q_handle, packed: *const u8, n: i64, block: c_int, format: c_int, scale_format: c_int, scales: *const c_void, out: *mut f32) -> i32;
    pub fn b2q_nf4_decode_f32(h: b2q_handle, packed: *const u8, nbytes: i64, block: c_int, absmaxs: *const f32, out: *mut f32) -> i32;
    pub fn b2q_nf4_encode_f32(h: b2q_handle, x: *const f32, n: i64, block: c_int, packed: *mut u8, absmaxs: *mut f32) -> i32;
    pub fn b2q_int8_quant_f32(h: b2q_handle, x: *const f32, n: i64, scale: f32, out: *mut i8) -> i32;
    pub fn b2q_int8_dequant_f32(h: b2q_handle, q: *const i8, n: i64, scale: f32, out: *mut f32) -> i32;
    pub fn b2q_distfp8_quantize_block_f32(h: b2q_handle, x: *const f32, n: i64, block: i64, q: *mut u8, absmaxs: *mut f32) -> i32;
    pub fn b2q_distfp8_dequantize_block_f32(h: b2q_handle, q: *const u8, n: i64, block: i64, absmaxs: *const f32, out: *mut f32) -> i32;
    pub fn b2q_rms_norm_quantize_fp8_bf16(h: b2q_handle, x_bf16: *const c_void, residual_bf16: *mut c_void, gamma_bf16: *const c_void, rows: i64, cols: i64, eps: f32, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8, y_out_bf16: *mut c_void) -> i32;
    pub fn b2q_rms_norm_quantize_fp8_block128_bf16(h: b2q_handle, x_bf16: *const c_void, residual_bf16: *mut c_void, gamma_bf16: *const c_void, rows: i64, cols: i64, eps: f32, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8, y_out_bf16: *mut c_void) -> i32;
    pub fn b2q_swiglu_quantize_fp8_block128_bf16(h: b2q_handle, gate: *const c_void, up: *const c_void, rows: i64, cols: i64, ld: i64, fmt: c_int, rounding: c_int, scales: *mut f32, codes: *mut u8) -> i32;
    pub fn b2q_kv8_append_bf16(h: b2q_handle, k: *const c_void, v: *const c_void, ld_k: i64, ld_v: i64, tokens: i64, q_starts: *const i32, seq_lens: *const i32, block_tables: *const i32, seqs: i64, table_width: i64, num_pages: i64, page_size: i64, n_kv_heads: i64, head_dim: i64, k_codes: *mut u8, v_codes: *mut u8, k_scales: *mut u8, v_scales: *mut u8) -> i32;
    pub fn b2q_kv8_attention_bf16(h: b2q_handle, q: *const c_void, ld_q: i64, tokens: i64, n_heads: i64, q_starts: *const i32, seq_lens: *const i32, block_tables: *const i32, seqs: i64, table_width: i64, num_pages: i64, page_size: i64, n_kv_heads: i64, head_dim: i64, k_codes: *const u8, v_codes: *const u8, k_scales: *const u8, v_scales: *const u8, scale: f32, window: i64, out: *mut c_void, lse: *mut f32) -> i32;
    pub fn b2q_kv_cache_quantize_f32(h: b2q_handle, x: *const f32, n_tokens: i64, head_dim: i64, bits: c_int, axis: c_int, codes: *mut u8, scales: *mut f32, zero_points: *mut f32) -> i32;
    pub fn b2q_kv_cache_quantize_bf16(h: b2q_handle, x_bf16: *const c_void, n_tokens: i64, head_dim: i64, bits: c_int, axis: c_int, codes: *mut u8, scales: *mut f32, zero_points: *mut f32) -> i32;
    pub fn b2q_kv_cache_dequantize_f32(h: b2q_handle, codes: *const u8, n_tokens: i64, head_dim: i64, axis: c_int, scales: *const f32, zero_points: *const f32, out: *mut f32) -> i32;
    pub fn b2q_kv_cache_dequantize_bf16(h: b2q_handle, codes: *const u8, n_tokens: i64, head_dim: i64, axis: c_int, scales: *const f32, zero_points: *const f32, out_bf16: *mut c_void) -> i32;
    pub fn b2q_kv_quantize_tokens_f32(h: b2q_handle, x: *const f32, n_tokens: i64, d: i64, bits: c_int, symmetric: c_int, codes: *mut u8, scales: *mut f32, zero_points: *mut f32) -> i32;
    pub fn b2q_kv_quantize_tokens_bf16(h: b2q_handle, x_bf16: *const c_void, n_tokens: i64, d: i64, bits: c_int, symmetric: c_int, codes: *mut u8, scales: *mut f32, zero_points: *mut f32) -> i32;
    pub fn b2q_kv_dequantize_tokens_f32(h: b2q_handle, codes: *const u8, n_tokens: i64, d: i64, symmetric: c_int, scales: *const f32, zero_points: *const f32, out: *mut f32) -> i32;
    pub fn b2q_kv_dequantize_tokens_bf16(h: b2q_handle, codes: *const u8, n_tokens: i64, d: i64, symmetric: c_int, scales: *const f32, zero_points: *const f32, out_bf16: *mut c_void) -> i32;
    pub fn b2q_dnn_quantize_to_fp8_f32(h: b2q_handle, x: *const f32, n: i64, codes: *mut u8, scale: *mut f32) -> i32;
    pub fn b2q_dnn_dequantize_from_fp8_f32(h: b2q_handle, codes: *const u8, scale: *const f32, n: i64, out: *mut f32) -> i32;
    pub fn b2q_dnn_quantize_to_int8_f32(h: b2q_handle, x: *const f32, n: i64, q: *mut i8, scale: *mut f32) -> i32;
    pub fn b2q_dnn_dequantize_from_int8_f32(h: b2q_handle, q: *const i8, scale: *const f32, n: i64, out: *mut f32) -> i32;
    pub fn b2q_dnn_quantize_block_scaled_f32(h: b2q_handle, x: *const f32, n: i64, block_size: u32, out: *mut u8, scales: *mut f32) -> i32;
    pub fn b2q_block_int8_quantize_f32(h: b2q_handle, x: *const f32, n: i64, block_size: i64, q: *mut i8, scales: *mut f32) -> i32;
    pub fn b2q_block_int8_dequantize_f32(h: b2q_handle, q: *const i8, scales: *const f32, n: i64, block_size: i64, out: *mut f32) -> i32;
    pub fn b2q_block_absmax_scale_f32(h: b2q_handle, x: *const f32, n: i64, block_size: i64, max_val: f32, scales: *mut f32) -> i32;
    pub fn b2q_pack_int4(h: b2q_handle, values: *const i8, n: i64, packed: *mut u32) -> i32;
    pub fn b2q_unpack_int4(h: b2q_handle, packed: *const u32, words: i64, out: *mut i8) -> i32;
    pub fn b2q_gemm_int4_f32(h: b2q_handle, a_packed: *const u32, scales_f16: *const c_void, b: *const f32, c: *mut f32, m: i64, n: i64, k: i64, group_size: i64) -> i32;
    pub fn b2q_gemv_int4_wo(h: b2q_handle, packed: *const u32, scales_f16: *const c_void, group_size: i64, x_bf16: *const c_void, tokens: i64, n: i64, k: i64, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_llm_int8_linear_f32(h: b2q_handle, x: *const f32, w: *const f32, samples: i64, rows: i64, cols: i64, threshold: f32, row_wise: c_int, out: *mut f32, wq: *mut i8, sw: *mut f32, xq: *mut i8, sx: *mut f32, acc: *mut i32, n_outliers: *mut i32) -> i32;
    pub fn b2q_gemm_i8(h: b2q_handle, a: *const i8, b: *const i8, M: i64, N: i64, K: i64, c_s32: *mut i32, c_f32: *mut f32, scale_a: *const f32, scale_b: *const f32) -> i32;
    pub fn b2q_gemm_fp8(h: b2q_handle, a: *const u8, w: *const u8, M: i64, N: i64, K: i64, fmt: c_int, scale_a: *const f32, scale_a_kind: c_int, scale_w: *const f32, scale_w_kind: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_gemm_fp8_ex(h: b2q_handle, d: *const b2q_gemm_fp8_desc) -> i32;
    pub fn b2q_gemm_fp8_block128(h: b2q_handle, a: *const u8, w: *const u8, M: i64, N: i64, K: i64, fmt: c_int, scale_a: *const f32, scale_w: *const f32, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_gemm_fp8_simt(h: b2q_handle, a: *const u8, w: *const u8, M: i64, N: i64, K: i64, fmt: c_int, decode_mode: c_int, scale_a: *const f32, scale_a_kind: c_int, scale_w: *const f32, scale_w_kind: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_tp_unique_id(id128: *mut u8) -> i32;
    pub fn b2q_tp_comm_init(id128: *const u8, tp: c_int, rank: c_int, nccl_comm: *mut *mut c_void) -> i32;
    pub fn b2q_tp_comm_destroy(nccl_comm: *mut c_void) -> i32;
    pub fn b2q_tp_create(h: b2q_handle, nccl_comm: *mut c_void, tp: c_int, rank: c_int, out: *mut b2q_tp) -> i32;
    pub fn b2q_tp_destroy(t: b2q_tp) -> i32;
    pub fn b2q_tp_exchange_buffer(t: b2q_tp, ptr: *mut *mut c_void, ipc_handle64: *mut u8) -> i32;
    pub fn b2q_tp_attach_peers(t: b2q_tp, ipc_handles: *const u8, direct_ptrs: *const *mut c_void) -> i32;
    pub fn b2q_gemm_fp8_scatter(h: b2q_handle, a: *const u8, w: *const u8, M: i64, N: i64, K: i64, fmt: c_int, scale_a: *const f32, scale_w: *const f32, bias: *const f32, inbox: *const *mut c_void, tp: c_int, rank: c_int) -> i32;
    pub fn b2q_tp_set_chunks(t: b2q_tp, chunks: c_int) -> i32;
    pub fn b2q_tp_plan(tp: c_int, peers_attached: c_int, tokens: i64, out_features: i64, mode: *mut c_int, chunks: *mut c_int) -> i32;
    pub fn b2q_tp_all_reduce_f32_to_bf16(t: b2q_tp, partial: *const f32, n: i64, y_bf16: *mut c_void) -> i32;
    pub fn b2q_tp_all_reduce_bf16(t: b2q_tp, y_bf16: *mut c_void, n: i64) -> i32;
    pub fn b2q_column_linear_forward(t: b2q_tp, x_codes: *const u8, x_scales: *const f32, w_codes: *const u8, w_scales: *const f32, bias: *const f32, tokens: i64, in_features: i64, out_local: i64, y_local: *mut c_void, y_gathered: *mut c_void) -> i32;
    pub fn b2q_row_linear_forward_allreduce(t: b2q_tp, x_codes: *const u8, x_scales: *const f32, w_codes: *const u8, w_scales: *const f32, bias: *const f32, tokens: i64, in_local: i64, out_features: i64, y: *mut c_void) -> i32;
    pub fn b2q_mlp_swiglu_fp8_forward(t: b2q_tp, x_bf16: *const c_void, w_gate_up: *const u8, s_gate_up: *const f32, w_down: *const u8, s_down: *const f32, tokens: i64, hidden: i64, ffn_local: i64, rounding: c_int, y_bf16: *mut c_void) -> i32;
    pub fn b2q_mlp_swiglu_fp8_forward_ex(t: b2q_tp, x_bf16: *const c_void, w_gate_up: *const u8, s_gate_up: *const f32, w_down: *const u8, s_down: *const f32, tokens: i64, hidden: i64, ffn_local: i64, rounding: c_int, gate_up_layout: c_int, y_bf16: *mut c_void) -> i32;
    pub fn b2q_interleave_rows128(h: b2q_handle, a: *const c_void, b: *const c_void, rows: i64, row_bytes: i64, out: *mut c_void) -> i32;
    pub fn b2q_grouped_gemm_fp8(h: b2q_handle, problems: *const b2q_gemm_fp8_problem, count: c_int, fmt: c_int, out_type: c_int) -> i32;
    pub fn b2q_grouped_gemm_fp8_rows(h: b2q_handle, a: *const u8, scale_a: *const f32, w: *const u8, scale_w: *const f32, row_offsets: *const i32, row_counts: *const i32, groups: c_int, capacity_rows: i64, N: i64, K: i64, fmt: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_ep_token_scatter(h: b2q_handle, in_: *const c_void, token: *const i32, slot: *const i32, pairs: i64, row_bytes: i64, expert_buf: *mut c_void) -> i32;
    pub fn b2q_ep_token_gather_bf16(h: b2q_handle, expert_out: *const c_void, slot: *const i32, weight: *const f32, tokens: i64, top_k: c_int, hidden: i64, out: *mut c_void) -> i32;
    pub fn b2q_moe_route_topk(h: b2q_handle, logits: *const f32, tokens: i64, n_experts: c_int, top_k: c_int, expert_idx: *mut i32, weight: *mut f32) -> i32;
    pub fn b2q_moe_assign_slots(h: b2q_handle, expert_idx: *const i32, pairs: i64, first_local: c_int, n_local: c_int, counts: *mut i32, offsets: *mut i32, slot_of_pair: *mut i32) -> i32;
    pub fn b2q_moe_scatter(h: b2q_handle, x: *const c_void, slot_of_pair: *const i32, pairs: i64, top_k: c_int, row_bytes: i64, expert_buf: *mut c_void) -> i32;
    pub fn b2q_moe_forward(t: b2q_tp, x_bf16: *const c_void, logits: *const f32, w_gate_up: *const u8, s_gate_up: *const f32, w_down: *const u8, s_down: *const f32, tokens: i64, hidden: i64, ffn: i64, n_experts: c_int, top_k: c_int, rounding: c_int, y_bf16: *mut c_void, counts_out: *mut i32) -> i32;
    pub fn b2q_moe_forward_fp4(t: b2q_tp, x_bf16: *const c_void, logits: *const f32, c_gate_up: *const u8, s_gate_up: *const u8, c_down: *const u8, s_down: *const u8, tokens: i64, hidden: i64, ffn: i64, n_experts: c_int, top_k: c_int, act_mode: c_int, y_bf16: *mut c_void, counts_out: *mut i32) -> i32;
    pub fn b2q_moe_forward_ex(t: b2q_tp, x_bf16: *const c_void, logits: *const f32, w_gate_up: *const u8, s_gate_up: *const f32, w_down: *const u8, s_down: *const f32, tokens: i64, hidden: i64, ffn: i64, n_experts: c_int, top_k: c_int, rounding: c_int, gate_up_layout: c_int, y_bf16: *mut c_void, counts_out: *mut i32) -> i32;
    pub fn b2q_gemv_fp4_wo(h: b2q_handle, codes: *const u8, scales: *const c_void, scale_format: c_int, block: c_int, x_bf16: *const c_void, tokens: i64, N: i64, K: i64, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_gemm_fp4_wo(h: b2q_handle, codes: *const u8, scales: *const c_void, scale_format: c_int, block: c_int, format: c_int, x_bf16: *const c_void, tokens: i64, N: i64, K: i64, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_gemm_fp4_blockscaled(h: b2q_handle, codes: *const u8, scales_e8m0: *const u8, x_bf16: *const c_void, tokens: i64, N: i64, K: i64, act_mode: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_grouped_gemm_fp4_rows(h: b2q_handle, codes: *const u8, scales_e8m0: *const u8, x_bf16: *const c_void, row_offsets: *const i32, groups: c_int, capacity_rows: i64, N: i64, K: i64, act_mode: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_ggml_block_bytes(type_: c_int) -> i64;
    pub fn b2q_ggml_block_size(type_: c_int) -> i64;
    pub fn b2q_ggml_quantize_f32(h: b2q_handle, type_: c_int, w: *const f32, n: i64, blocks: *mut u8) -> i32;
    pub fn b2q_ggml_dequantize(h: b2q_handle, type_: c_int, blocks: *const u8, n: i64, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_wq_packed_words(rows: i64, cols: i64, bits: c_int) -> i64;
    pub fn b2q_gptq_quantize_f32(h: b2q_handle, weight: *const f32, hessian_diag: *const f32, rows: i64, cols: i64, group_size: i64, bits: c_int, symmetric: c_int, packed: *mut u32, scales: *mut f32) -> i32;
    pub fn b2q_wq_dequantize(h: b2q_handle, packed: *const u32, scales: *const f32, zeros: *const f32, rows: i64, cols: i64, group_size: i64, bits: c_int, out: *mut c_void, out_type: c_int) -> i32;
    pub fn b2q_awq_scale_search_f32(h: b2q_handle, act_stats: *const f32, num_channels: i64, scale_out: *mut f32) -> i32;
    pub fn b2q_awq_quantize_f32(h: b2q_handle, weight: *const f32, channel_scales: *const f32, group_scales: *const f32, rows: i64, cols: i64, group_size: i64, bits: c_int, packed: *mut u32, zeros: *mut f32) -> i32;
    pub fn b2q_fused_dequant_gemv_f32(h: b2q_handle, packed: *const u32, scales: *const f32, zeros: *const f32, x: *const f32, rows: i64, cols: i64, group_size: i64, bits: c_int, split_k: c_int, y: *mut f32) -> i32;
    pub fn b2q_classify_workload(m: u32, n: u32, k: u32) -> i32;
    pub fn b2q_ref_tile_config(dtype: c_int, m: u32, n: u32, k: u32, out: *mut b2q_tile_config) -> i32;
    pub fn b2q_fp8_compute_split_k(m: u32, n: u32, k: u32) -> u32;
    pub fn b2q_select_tile(dtype: c_int, m: u32, n: u32, k: u32, out: *mut b2q_tile_config, kernel_id: *mut c_int) -> i32;
}
