/* Prints sizeof / offsetof of the rotary and block operators' C-ABI structs so that
 * tests/test_attn_ops.py can compare them with the ctypes mirrors in shrimp/_lib.py. */
#include <stddef.h>
#include <stdio.h>

#include "shrimp_hip.h"

#define F(S, f) printf("%s.%s %zu\n", #S, #f, offsetof(S, f))
#define Z(S) printf("%s.__size__ %zu\n", #S, sizeof(S))

int main(void) {
  Z(shrimp_rope_args);
  F(shrimp_rope_args, q); F(shrimp_rope_args, k); F(shrimp_rope_args, q_sb);
  F(shrimp_rope_args, q_sh); F(shrimp_rope_args, q_sn); F(shrimp_rope_args, k_sb);
  F(shrimp_rope_args, k_sh); F(shrimp_rope_args, k_sn); F(shrimp_rope_args, pos);
  F(shrimp_rope_args, p_sb); F(shrimp_rope_args, p_sn); F(shrimp_rope_args, p_sa);
  F(shrimp_rope_args, freqs); F(shrimp_rope_args, q_w); F(shrimp_rope_args, k_w);
  F(shrimp_rope_args, q_out); F(shrimp_rope_args, k_out); F(shrimp_rope_args, gq);
  F(shrimp_rope_args, gk); F(shrimp_rope_args, gq_sb); F(shrimp_rope_args, gq_sh);
  F(shrimp_rope_args, gq_sn); F(shrimp_rope_args, gk_sb); F(shrimp_rope_args, gk_sh);
  F(shrimp_rope_args, gk_sn); F(shrimp_rope_args, B); F(shrimp_rope_args, S);
  F(shrimp_rope_args, H); F(shrimp_rope_args, Hk); F(shrimp_rope_args, D);
  F(shrimp_rope_args, axes); F(shrimp_rope_args, sections); F(shrimp_rope_args, dt);
  F(shrimp_rope_args, pos_dt); F(shrimp_rope_args, freq_f64); F(shrimp_rope_args, w_dt);
  F(shrimp_rope_args, interleaved); F(shrimp_rope_args, inverse); F(shrimp_rope_args, eps);
  Z(shrimp_block_select_args);
  F(shrimp_block_select_args, q); F(shrimp_block_select_args, q_sb);
  F(shrimp_block_select_args, q_sh); F(shrimp_block_select_args, q_sn);
  F(shrimp_block_select_args, means); F(shrimp_block_select_args, q_lens);
  F(shrimp_block_select_args, k_lens); F(shrimp_block_select_args, sel);
  F(shrimp_block_select_args, B); F(shrimp_block_select_args, H);
  F(shrimp_block_select_args, Hk); F(shrimp_block_select_args, Sq);
  F(shrimp_block_select_args, Sk); F(shrimp_block_select_args, D);
  F(shrimp_block_select_args, block); F(shrimp_block_select_args, topk);
  F(shrimp_block_select_args, dt);
  Z(shrimp_attn_blocks_args);
  F(shrimp_attn_blocks_args, q); F(shrimp_attn_blocks_args, k); F(shrimp_attn_blocks_args, v);
  F(shrimp_attn_blocks_args, q_sb); F(shrimp_attn_blocks_args, q_sh);
  F(shrimp_attn_blocks_args, q_sn); F(shrimp_attn_blocks_args, k_sb);
  F(shrimp_attn_blocks_args, k_sh); F(shrimp_attn_blocks_args, k_sn);
  F(shrimp_attn_blocks_args, v_sb); F(shrimp_attn_blocks_args, v_sh);
  F(shrimp_attn_blocks_args, v_sn); F(shrimp_attn_blocks_args, sel);
  F(shrimp_attn_blocks_args, q_lens); F(shrimp_attn_blocks_args, k_lens);
  F(shrimp_attn_blocks_args, out); F(shrimp_attn_blocks_args, lse);
  F(shrimp_attn_blocks_args, B); F(shrimp_attn_blocks_args, H);
  F(shrimp_attn_blocks_args, Hk); F(shrimp_attn_blocks_args, Sq);
  F(shrimp_attn_blocks_args, Sk); F(shrimp_attn_blocks_args, d);
  F(shrimp_attn_blocks_args, block); F(shrimp_attn_blocks_args, topk);
  F(shrimp_attn_blocks_args, dt); F(shrimp_attn_blocks_args, scale);
  Z(shrimp_attn_blocks_grads);
  F(shrimp_attn_blocks_grads, g); F(shrimp_attn_blocks_grads, g_sb);
  F(shrimp_attn_blocks_grads, g_sh); F(shrimp_attn_blocks_grads, g_sn);
  F(shrimp_attn_blocks_grads, g_lse); F(shrimp_attn_blocks_grads, dq);
  F(shrimp_attn_blocks_grads, dk); F(shrimp_attn_blocks_grads, dv);
  F(shrimp_attn_blocks_grads, workspace); F(shrimp_attn_blocks_grads, workspace_bytes);
  return 0;
}
