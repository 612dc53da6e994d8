/*
 * hive_gpu.h -- C-ABI of libhive_gpu.so, the MI355X (gfx950) batched Hive
 * engine.  This is the drop-in boundary: the Python package
 * hive_neuralnet_amd.hive_gpu (the counterpart of the reference's
 * hive_gpu.load_extension()) binds these symbols with ctypes; any other FFI
 * can bind them the same way.
 *
 * Conventions (all entry points):
 *   - pointers are device pointers; the caller allocates every input and
 *     output (the reference allocates outputs inside its wrappers -- the
 *     Python layer does that here, with the reference's fill values);
 *   - `stream` is a hipStream_t (void* so this header needs no HIP headers);
 *     work is enqueued on it and the call returns without synchronising;
 *   - the return value is a hipError_t code (0 = success) of the launch;
 *   - sizes <= 0 are a no-op returning 0;
 *   - byte formats are the reference's: a state row is 3424 bytes
 *     (HiveState, hive_gpu/csrc/hive_state.cuh:239-269), a move is 6 bytes
 *     {u8 type, u8 piece_type, u16 from, u16 to} (hive_state.cuh:228-233),
 *     legal lists are [B, 256, 6] with zero padding, features are [B, 122].
 *
 * Each declaration names the reference interface it replaces
 * (chrismejias/hive_neuralnet, file:line).
 */
#ifndef HIVE_GPU_H
#define HIVE_GPU_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HG_ABI_VERSION 1
#define HG_STATE_BYTES 3424
#define HG_MOVE_BYTES 6
#define HG_MAX_LEGAL_MOVES 256
#define HG_FNN_FEAT_DIM 122

int hg_abi_version(void);

/* initialize_tables -- hive_gpu/csrc/game_logic.cu:404-407, bindings.cpp:257.
 * The hex tables are closed-form constants here; kept for API parity. */
int hg_initialize_tables(void);

/* create_initial_states -- game_logic.cu:413-428 (init_states_kernel :54-59).
 * Writes every byte of states[B][3424]. */
int hg_create_initial_states(uint8_t* states, int64_t B, int expansion_mask, void* stream);

/* apply_moves_batch -- game_logic.cu:465-477 (apply_moves_kernel :233-242).
 * moves[B][6]; states updated in place. */
int hg_apply_moves(uint8_t* states, const uint8_t* moves, int64_t B, void* stream);

/* check_results_batch -- game_logic.cu:483-497.  results[B] int32. */
int hg_check_results(const uint8_t* states, int64_t B, int32_t* results, void* stream);

/* generate_legal_moves_batch -- game_logic.cu:436-459.
 * moves[B][256][6] (fully written, zero padded), num_legal[B]. */
int hg_generate_legal_moves(const uint8_t* states, int64_t B, uint8_t* moves, int32_t* num_legal, void* stream);

/* generate_legal_moves_and_fnn_features_batch -- game_logic.cu:1439-1464. */
int hg_generate_legal_moves_and_fnn_features(const uint8_t* states, int64_t B, uint8_t* moves,
                                             int32_t* num_legal, float* features, void* stream);

/* Fused move generation + FNN features + action indices in one pass: the
 * outputs of generate_legal_moves_and_fnn_features_batch (game_logic.cu:1439)
 * followed by legal_moves_to_actions_batch (game_logic.cu:837) without the
 * list round trip through HBM.  actions[B][256] int32, -1 padded.  No single
 * reference entry point; same spirit as the reference's own fused
 * mcts_select_replay_legal_fnn_root_slots_batch. */
int hg_legal_features_actions(const uint8_t* states, int64_t B, uint8_t* moves, int32_t* num_legal,
                              float* features, int32_t* actions, void* stream);

/* hg_legal_features_actions taking the positions in buckets of 4 turns,
 * latest first (a wave's cost is its longer position; the launch ends with
 * its longest waves): identical outputs.  workspace:
 * hg_legal_features_actions_ordered_workspace(B) bytes, 4-byte aligned: two
 * arrays of 32 bucket counts, then one index list per bucket.  A call needs
 * counts[parity] zero, uses it and clears counts[parity ^ 1]: zero-fill a new
 * workspace once, then alternate parity (0, 1, 0, ...) on calls that use it
 * on one stream.  A HIP graph replays the parity it captured and would count
 * into arrays that nothing clears: capture hg_legal_features_actions instead
 * (the Python mirror does so while its stream is capturing).  No reference
 * counterpart (same outputs as the entry above). */
int64_t hg_legal_features_actions_ordered_workspace(int64_t B);
int hg_legal_features_actions_ordered(const uint8_t* states, int64_t B, uint8_t* moves, int32_t* num_legal,
                                      float* features, int32_t* actions, void* workspace, int parity,
                                      void* stream);

/* extract_fnn_features_batch -- game_logic.cu:1409-1431.
 * features for caller-supplied lists (num_legal clamped to [0, 256]). */
int hg_extract_fnn_features(const uint8_t* states, const uint8_t* moves, const int32_t* num_legal, int64_t B,
                            float* features, void* stream);

/* legal_moves_to_actions_batch -- game_logic.cu:837-857.
 * actions[B][256] int32: action index per listed move, -1 beyond num_legal
 * and for moves outside the 17x17 window around the centroid. */
int hg_legal_moves_to_actions(const uint8_t* states, const uint8_t* moves, const int32_t* num_legal, int64_t B,
                              int32_t* actions, void* stream);

/* compute_centroids_batch -- game_logic.cu:910-926.  centroids[B][2] int32. */
int hg_compute_centroids(const uint8_t* states, int64_t B, int32_t* centroids, void* stream);

/* fnn_successor_features_batch -- game_logic.cu:1648-1671.
 * For i < N: features[i] of states[action_to_root[i]] after
 * legal_moves[action_to_root[i]][move_indices[i]], with the compact
 * successor move summary (move_gen.cuh:1416-1563).  num_roots is the row
 * count of states/legal_moves; rows whose root or move index is out of range
 * get all-zero features (the reference reads out of bounds there). */
int hg_fnn_successor_features(const uint8_t* states, const uint8_t* legal_moves, int64_t num_roots,
                              const int64_t* action_to_root, const int64_t* move_indices, int64_t N, float* features,
                              void* stream);

/* hg_fnn_leaf_eval -- FNN leaf evaluation, fused (restates the torch chain of
 * the reference's FNNMCTSOrchestrator._eval_states,
 * hive_fnn/fnn_mcts_orchestrator.py:243-316, over HiveFNN.encode / value_head /
 * score_actions, hive_fnn/fnn_network.py:175-220; the reference has no kernel
 * for it).  Network widths: hidden = embedding = action tower = 64, F <= 128
 * features (even).  Weights are the nn.Linear / nn.LayerNorm tensors as
 * stored (row-major [out][in]).
 *
 * features[T + N][F]: the T leaf rows, then the successor rows; the
 * successor rows of leaf t are T + offsets[t] .. + num_legal[t], and
 * succ_leaf[i] = t for successor row i (i < N).  With
 *   e(x)          = fc2(LayerNorm(sigmoid(fc1 x)))     (eps 1e-5)
 *   root_values[t] = tanh(value_w . e(leaf t) + value_b)
 *   child_q[t][i]  = -tanh(value_w . e(successor i of t) + value_b)
 *   logit_i        = action2_w . sigmoid(action1_w [e(leaf t) | e(succ i)]
 *                                        + action1_b) + action2_b
 *   priors[t][i]   = softmax over i < num_legal[t] of logit_i
 * priors and child_q are [T][256], zero beyond num_legal[t].
 * workspace: T * 64 + 2 * N floats, 16-byte aligned (the root half of the
 * action tower per leaf, then logits and child values per successor row);
 * features must be 8-byte aligned.  Returns hipErrorInvalidValue for other
 * shapes or alignments. */
int hg_fnn_leaf_eval(const float* features, int64_t T, int64_t N, int F, const int64_t* offsets,
                     const int32_t* num_legal, const int64_t* succ_leaf, const float* fc1_w, const float* fc1_b,
                     const float* ln_w, const float* ln_b, const float* fc2_w, const float* fc2_b,
                     const float* value_w, float value_b, const float* action1_w, const float* action1_b,
                     const float* action2_w, float action2_b, float* workspace, float* priors, float* root_values,
                     float* child_q, void* stream);

/* root_tactical_probe_batch -- game_logic.cu:1579-1616 (root_tactical_probe_kernel
 * :290-397; has_immediate_surround_win_for_current_player and
 * generate_non_decreasing_surround_replies, move_gen.cuh:825-898).  For each
 * root: winning[B] int64 = the immediate win with the highest prior (first on
 * ties; only when the opponent's queen has 5 neighbours), else the lowest
 * slot after which every reply loses at once (opponent queen at 4 or 5),
 * else -1; allowed[B][256] uint8 = legal slots, minus those after which the
 * opponent wins at once (only when the own queen has 5 neighbours);
 * forced[B] uint8 = that screen left no slot.  num_legal is clamped to 256.
 * workspace: hg_root_tactical_probe_workspace(B) int32, 8-byte aligned (job
 * counters, job lists, the two-move candidates' failure flags and their
 * grandchildren's list).  Six launches on `stream`, no host
 * synchronisation. */
int64_t hg_root_tactical_probe_workspace(int64_t B);
int hg_root_tactical_probe(const uint8_t* states, const uint8_t* legal_moves, const int32_t* num_legal,
                           const float* priors, int64_t B, int enable_win_in_one, int enable_check_opponent_wins,
                           int enable_win_in_two, int64_t* winning, uint8_t* allowed, uint8_t* forced,
                           int32_t* workspace, void* stream);

/* hg_root_tactical_probe with no workspace argument and no allocation.  No
 * counterpart in the reference: it is for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).  The job lists live in a static device array of this
 * library, one per GPU, sized for at most HG_PROBE_NOALLOC_MAX_ROOTS roots
 * (25.2 MB); B above that returns hipErrorInvalidValue and launches nothing.
 * Every call on one GPU shares that GPU's array: calls that overlap on one
 * GPU (other streams, other threads) race and must be serialised by the
 * caller (the Python binding orders its own calls on one GPU by an event,
 * outside graph capture).  Outputs as hg_root_tactical_probe.
 * hg_probe_scratch_init looks up the current device's array address (the
 * first call on a device does it too) and keeps it for the process; after a
 * hipDeviceReset that address is stale: call hg_probe_scratch_init again on
 * that device, with it current, before the next hg_root_tactical_probe_noalloc. */
#define HG_PROBE_NOALLOC_MAX_ROOTS 4096
int hg_probe_scratch_init(void);
int hg_root_tactical_probe_noalloc(const uint8_t* states, const uint8_t* legal_moves, const int32_t* num_legal,
                                   const float* priors, int64_t B, int enable_win_in_one,
                                   int enable_check_opponent_wins, int enable_win_in_two, int64_t* winning,
                                   uint8_t* allowed, uint8_t* forced, void* stream);

/* generate_legal_mask_batch / generate_legal_moves_and_mask_batch --
 * game_logic.cu:737-806 (legal_mask_kernel, state_encoder.cuh:908-976).
 * masks[B][85834] f32 (written whole): 1.0 at the action index of every
 * legal slot whose cells fall in the 17x17 window around the centroid, and at
 * PASS_ACTION_INDEX for a PASS.  moves[B][256][6], num_legal[B] as
 * hg_generate_legal_moves; actions[B][256] int32 is scratch (the slots'
 * action indices). */
int hg_legal_mask(const uint8_t* states, int64_t B, uint8_t* moves, int32_t* num_legal, int32_t* actions,
                  float* masks, void* stream);

/* Successor rows of a batch of leaves with the row count kept on the device
 * (no counterpart in the reference, which sizes them on the host:
 * fnn_mcts_orchestrator.py:243-316): offsets[T] int64 = exclusive prefix of
 * the clamped num_legal, total int64 = their sum, the row map (leaf, slot) and
 * features[total][122] of every successor in (leaf, slot) order
 * (fnn_successor_features_kernel semantics, game_logic.cu:182-229).  features
 * must hold T * 256 rows; workspace hg_successor_rows_workspace(T) bytes,
 * 8-byte aligned: offsets, total, then the map. */
int64_t hg_successor_rows_workspace(int64_t T);
int hg_successor_rows(const uint8_t* states, const uint8_t* legal_moves, const int32_t* num_legal, int64_t T,
                      void* workspace, float* features, void* stream);
/* hg_successor_rows in its two steps, for a caller that sizes the features by
 * the total between them: the plan (offsets, total, map into the workspace),
 * then the planned rows' features (`total` rows of 122). */
int hg_successor_plan(const int32_t* num_legal, int64_t T, void* workspace, void* stream);
int hg_successor_planned_rows(const uint8_t* states, const uint8_t* legal_moves, int64_t T, void* workspace,
                              float* features, void* stream);

/* hg_fnn_leaf_eval over the leaves' own legal lists, with no host
 * synchronisation: hg_successor_rows into the workspace, then the network
 * (F = 122; the root rows are root_features [T][122]).  Outputs as
 * hg_fnn_leaf_eval.  workspace: hg_fnn_leaf_eval_lists_workspace(T, F) bytes,
 * 256-byte aligned (the successor rows at capacity T * 256). */
int64_t hg_fnn_leaf_eval_lists_workspace(int64_t T, int F);
int hg_fnn_leaf_eval_lists(const uint8_t* leaf_states, const uint8_t* legal_moves, const int32_t* num_legal,
                           const float* root_features, int64_t T, int F, const float* fc1_w, const float* fc1_b,
                           const float* ln_w, const float* ln_b, const float* fc2_w, const float* fc2_b,
                           const float* value_w, float value_b, const float* action1_w, const float* action1_b,
                           const float* action2_w, float action2_b, void* workspace, float* priors,
                           float* root_values, float* child_q, void* stream);

/* queen_escape_flags_batch -- game_logic.cu:1538-1554.  flags[B] uint8. */
int hg_queen_escape_flags(const uint8_t* states, int64_t B, uint8_t* flags, void* stream);

/* The Gumbel root candidates with their reserve slots, in one launch
 * (FNNMCTSOrchestrator._root_candidate_slots with reserve > 0,
 * hive_fnn/fnn_mcts_orchestrator.py:338-444, there a chain of torch ops over
 * a copy of every child state).  Legal slot j of root r qualifies when its
 * move raises the surround count of the opponent's queen (occupied on-grid
 * neighbours of its cell, 0 while it is unplaced) and, when immobile_only !=
 * 0, the child's side to move has no queen escape (queen_escape_flags_batch
 * on the child).  qualifies (optional): [B][256] uint8, 1 / 0, all 256 slots
 * written.  candidates (optional, then priors [B][256] f32 required):
 * [B][k] int32, columns 0 .. reserve-1 the qualifying slots by prior (-1
 * past their count, at most `reserve`), columns reserve .. k-1 the slots
 * that are legal, allowed (allowed [B][256] uint8, or NULL: all) and not
 * reserved, by prior, followed by the others (ranked at -1e30); every ranking
 * stable (ties to the lower slot).  num_legal is clamped to [0, 256];
 * 1 <= k <= 256, 0 <= reserve <= k. */
int hg_reserve_candidates(const uint8_t* states, const uint8_t* legal_moves, const int32_t* num_legal,
                          const uint8_t* allowed, const float* priors, int64_t B, int k, int reserve,
                          int immobile_only, uint8_t* qualifies, int32_t* candidates, void* stream);

/* The candidate rows of hg_reserve_candidates from given masks: qualifies and
 * valid [B][256] uint8 (nonzero = set), priors [B][256] f32 -> candidates
 * [B][k] int32 (FNNMCTSOrchestrator._root_candidate_slots from its qualifying
 * mask, fnn_mcts_orchestrator.py:411-444). */
int hg_candidate_rows(const uint8_t* qualifies, const uint8_t* valid, const float* priors, int64_t B, int k,
                      int reserve, int32_t* candidates, void* stream);

/* One ply of seeded random play (the position generator of the benchmark
 * configurations; no reference counterpart -- the reference's own pattern is
 * torch.rand x n_legal + apply_moves_batch, hive_gpu/endgame_generator.py:268-276).
 * Game i is active while ply < target_i and its result is 0, where target_i =
 * Philox4x32-10(key=(seed,0), ctr=(i,0,0,0))[0] mod (max_ply+1), or max_ply
 * when lockstep != 0.  An active game applies
 * moves[i][(Philox(key, (i,ply+1,0,0))[0] * num_legal[i]) >> 32] and, when
 * plies_done is not NULL, increments plies_done[i]. */
int hg_random_play_step(uint8_t* states, const uint8_t* moves, const int32_t* num_legal, int64_t B, int ply,
                        int max_ply, int lockstep, uint32_t seed, int32_t* plies_done, void* stream);

/* The plies 0 .. max_ply - 1 of hg_random_play_step (each after the legal
 * lists of hg_generate_legal_moves) in one launch, every game's board held in
 * LDS from its first ply to its last (the state rows receive each ply's
 * changed bytes): the same states and plies_done.  moves: scratch of
 * B * 256 * 6 bytes, required (its first aligned 4-byte word holds the
 * launch's counter of game pairs handed out; calls that share a scratch
 * buffer on different streams race); its contents afterwards are
 * unspecified.  No
 * reference counterpart (the generator of the benchmark configurations, as
 * hg_random_play_step). */
int hg_random_play(uint8_t* states, uint8_t* moves, int64_t B, int max_ply, int lockstep, uint32_t seed,
                   int32_t* plies_done, void* stream);

/* ---------------------------------------------------------------- MCTS tree
 * The reference's structure-of-arrays tree (mcts_tree.cuh:31-45), one pool of
 * max_nodes slots per game, arrays [B, max_nodes] (move_bytes [B, max_nodes, 6],
 * node_count [B]); child_init_q is the extra [B, max_nodes] array the
 * reference passes beside the struct.  Passed by host pointer.
 *
 * Order of effect: simulations of one game take effect in simulation-index
 * order (sim = k*B + game): each selection sees earlier selections' virtual
 * losses, the earliest simulation reaching an unexpanded leaf expands it,
 * node ids are handed out in that order, float updates happen in that order.
 * The reference applies the same updates with atomics in whatever order its
 * threads run. */
typedef struct hg_tree {
    int32_t* visit_count;
    float* total_value;
    float* prior;
    int32_t* parent_idx;
    float* virtual_q_penalty;
    uint8_t* move_bytes;
    int32_t* action_idx;
    int32_t* first_child;
    int32_t* num_children;
    int8_t* is_terminal;
    float* terminal_value;
    int32_t* node_count;
    float* child_init_q;
    int64_t max_nodes;
} hg_tree;

/* ---- legacy action-space engine (hive_gpu/gpu_native_mcts.py; the twelve
 * tree arrays only, no child_init_q).  Same canonical order as below. */

/* mcts_select_batch -- game_logic.cu:961-993 (mcts_select_kernel,
 * mcts_tree.cuh:205-296): PUCT from the root at every level, first maximum,
 * the first child when no score beats -1e30; virtual loss on every entered
 * node.  T = W * B, outputs as hg_mcts_select_root_slots. */
int hg_mcts_select(const hg_tree* tree, const int8_t* game_active, const int32_t* root_nodes, float c_puct, int64_t B,
                   int W, int32_t* leaf_idx, uint8_t* move_paths, int32_t* path_lens, int32_t* vl_paths,
                   int32_t* vl_lens, void* stream);

/* mcts_expand_batch -- game_logic.cu:1018-1045 (mcts_expand_kernel,
 * mcts_tree.cuh:330-433): children for the legal moves that have an action
 * index, prior = action_probs[sim][action] ([T][85834] f32); was_expanded[T]. */
int hg_mcts_expand(const hg_tree* tree, const int32_t* leaf_idx, const uint8_t* leaf_states, const uint8_t* legal_moves,
                   const int32_t* num_legal, const float* action_probs, const int32_t* results, int64_t B,
                   int64_t total, int8_t* was_expanded, void* stream);

/* mcts_backprop_batch -- game_logic.cu:1328-1349 (mcts_backprop_kernel,
 * mcts_tree.cuh:555-605). */
int hg_mcts_backprop(const hg_tree* tree, const int32_t* leaf_idx, const float* nn_values, const int32_t* vl_paths,
                     const int32_t* vl_lens, const int8_t* was_expanded, int64_t B, int64_t total, void* stream);

/* mcts_expand_and_backprop_batch -- game_logic.cu:1053-1080
 * (mcts_expand_and_backprop_kernel, mcts_tree.cuh:435-553). */
int hg_mcts_expand_backprop(const hg_tree* tree, const int32_t* leaf_idx, const uint8_t* leaf_states,
                            const uint8_t* legal_moves, const int32_t* num_legal, const float* action_probs,
                            const int32_t* results, const float* nn_values, const int32_t* vl_paths,
                            const int32_t* vl_lens, int64_t B, int64_t total, void* stream);

/* mcts_extract_policy_batch -- game_logic.cu:1355-1379
 * (mcts_extract_policy_kernel, mcts_tree.cuh:607-687): policies[B][85834]
 * f32, written whole: root visit counts (pruned below pruning_threshold x
 * the maximum, raised to 1/temperature, normalised; uniform when none),
 * one-hot on the most visited child once move_numbers[g] >= temp_drop_move. */
int hg_mcts_extract_policy(const hg_tree* tree, const int32_t* move_numbers, const int32_t* root_nodes,
                           float temperature, int temp_drop_move, float pruning_threshold, int64_t B, float* policies,
                           void* stream);

/* Hard tree rebase of FNNMCTSOrchestrator._reroot_tree
 * (hive_fnn/fnn_mcts_orchestrator.py:1122-1142, rebase_tree_each_move): for
 * each game g with reset[g] != 0, every node of the game's rows returns to
 * its initial fill (visit/value/prior/children/terminal/child_init_q 0,
 * parent/action/first_child -1, move bytes 0; virtual_q_penalty untouched,
 * as in the reference), node_count[g] = 1, root_node[g] = 0.  Only the used
 * prefix [0, node_count[g]) is written: the nodes beyond it still hold the
 * initial fill.  B <= 65535. */
int hg_mcts_reset_trees(const hg_tree* tree, const int8_t* reset, int32_t* root_node, int64_t B, void* stream);

/* mcts_select_with_root_slots_batch -- game_logic.cu:1134-1175
 * (mcts_select_with_root_slots_kernel, mcts_tree.cuh:811-955).
 * T = W * num_candidates * B simulations, sim = (w*C + c)*B + game.
 * Outputs, whole rows written (entries past path_lens / vl_lens are zero, as the
 * reference's zero-filled outputs): leaf_idx[T], move_paths[T][128][6],
 * path_lens[T], vl_paths[T][128], vl_lens[T]. */
int hg_mcts_select_root_slots(const hg_tree* tree, const int8_t* game_active, const int32_t* root_nodes,
                              const int32_t* root_slots, int num_candidates, int max_root_children, float c_puct,
                              int64_t B, int W, int deterministic_non_root, float non_root_sigma, float q_penalty,
                              int32_t* leaf_idx, uint8_t* move_paths, int32_t* path_lens, int32_t* vl_paths,
                              int32_t* vl_lens, void* stream);

/* mcts_select_with_root_mask_batch -- game_logic.cu:1088-1129
 * (mcts_select_with_root_mask_kernel, mcts_tree.cuh:689-800).  T = W * B. */
int hg_mcts_select_root_mask(const hg_tree* tree, const int8_t* game_active, const int32_t* root_nodes,
                             const int8_t* alive_mask, int max_root_children, float c_puct, int64_t B, int W,
                             int deterministic_non_root, float non_root_sigma, float q_penalty, int32_t* leaf_idx,
                             uint8_t* move_paths, int32_t* path_lens, int32_t* vl_paths, int32_t* vl_lens,
                             void* stream);

/* mcts_replay_batch -- game_logic.cu:1000-1015 (mcts_replay_kernel, mcts_tree.cuh:298-320).
 * leaf_states[s] = root_states[s % B] with the path moves applied; rows with
 * leaf_idx < 0 are left untouched. */
int hg_mcts_replay(const uint8_t* root_states, int64_t B, uint8_t* leaf_states, const uint8_t* move_paths,
                   const int32_t* path_lens, const int32_t* leaf_idx, int64_t total, void* stream);

/* The replay step of mcts_select_replay_legal_fnn_root_slots_batch
 * (game_logic.cu:1183-1254), which replays into a zero-filled buffer: as
 * hg_mcts_replay, and rows with leaf_idx < 0 are written as zero rows, so
 * leaf_states may start uninitialised. */
int hg_mcts_replay_fill(const uint8_t* root_states, int64_t B, uint8_t* leaf_states, const uint8_t* move_paths,
                        const int32_t* path_lens, const int32_t* leaf_idx, int64_t total, void* stream);

/* mcts_expand_dense_priors_batch -- game_logic.cu:1259-1288
 * (mcts_expand_dense_priors_kernel, mcts_tree.cuh:971-1062).  was_expanded[total] int8. */
int hg_mcts_expand_dense(const hg_tree* tree, const float* child_q_values, const int32_t* leaf_idx,
                         const uint8_t* leaf_states, const uint8_t* legal_moves, const int32_t* num_legal,
                         const float* priors_per_legal, const int32_t* results, int64_t B, int64_t total,
                         int8_t* was_expanded, void* stream);

/* mcts_expand_and_backprop_dense_priors_batch -- game_logic.cu:1293-1323
 * (mcts_expand_and_backprop_dense_priors_kernel, mcts_tree.cuh:1068-1187). */
int hg_mcts_expand_backprop_dense(const hg_tree* tree, const float* child_q_values, const int32_t* leaf_idx,
                                  const uint8_t* leaf_states, const uint8_t* legal_moves, const int32_t* num_legal,
                                  const float* priors_per_legal, const int32_t* results, const float* nn_values,
                                  const int32_t* vl_paths, const int32_t* vl_lens, float q_penalty, int64_t B,
                                  int64_t total, void* stream);

/* hg_mcts_expand_backprop_dense with a workspace of
 * hg_mcts_expand_backprop_dense_workspace(B, total) bytes (4-byte aligned;
 * accepted and not written: the plan lives in on-chip memory): the same
 * tree, the simulations of different root children applied in parallel (one
 * workgroup per game: a planning wave settles node ids and the root's
 * statistics in simulation order, then one wave per root child).  Identical
 * results; the
 * one-wave-per-game order is kept for games whose node pool could run short
 * or with a path that is not a selection path (each entry a node of the pool
 * whose parent is the entry before it, the last entry the leaf).  Path
 * entries are node ids below max_nodes, as in the reference. */
int64_t hg_mcts_expand_backprop_dense_workspace(int64_t B, int64_t total);
int hg_mcts_expand_backprop_dense_ws(const hg_tree* tree, const float* child_q_values, const int32_t* leaf_idx,
                                     const uint8_t* leaf_states, const uint8_t* legal_moves,
                                     const int32_t* num_legal, const float* priors_per_legal, const int32_t* results,
                                     const float* nn_values, const int32_t* vl_paths, const int32_t* vl_lens,
                                     float q_penalty, int64_t B, int64_t total, void* workspace, void* stream);

/* mcts_apply_root_noise -- game_logic.cu:1384-1402 (mcts_root_noise_kernel,
 * mcts_tree.cuh:1192-1234).  noise[B][max_children_pad]; children beyond the
 * pad are left unchanged (the reference reads past the row there). */
int hg_mcts_root_noise(const hg_tree* tree, const float* noise, const int32_t* root_nodes, int max_children_pad,
                       float dir_eps, float root_policy_temp, int64_t B, void* stream);

/* Search counters of one simulation wave (no counterpart in the reference:
 * instrumentation for throughput accounting).  Over rows t < total with
 * leaf_idx[t] >= 0: stats[0] += 1, stats[1] += num_legal[t], stats[2] +=
 * vl_lens[t]; and stats[3] += total.  stats is int64[4] in device memory,
 * updated in stream order (calls on one stream accumulate). */
int hg_mcts_wave_stats(const int32_t* leaf_idx, const int32_t* num_legal, const int32_t* vl_lens, int64_t total,
                       int64_t* stats, void* stream);

/* One decision of the Gumbel root search's sequential halving
 * (fnn_mcts_orchestrator.py:650-731: the statistics of the candidates' root
 * children, the batch-global sigma, the scores and the survivors; no single
 * reference entry point -- the reference runs these as torch ops between
 * rounds).  candidates[B][C] root slots (-1 = none), 1 <= C <= 64; base[B][256]
 * the Gumbel draw + legal logit of every slot.  A column's visits N and Q
 * (-W / max(N, 1) when N > root_q_min_visits, else 0) are those of the root
 * child in its slot (0, 0 outside the root's children); sigma = (c_visit + the
 * largest candidate N of the batch) * c_scale; score = base[g][slot] + sigma *
 * Q, -1e30 for an empty column.  keep > 0 (= C / 2 between rounds): the
 * columns in descending score order (ties to the lower column), the first
 * keep written to cand_out[B][keep] -- the first max(1, nonempty / 2) as
 * their slots, the rest -1.  keep = 0 (the final choice): chosen[g] = the
 * slot of the first highest column, 0 when it is empty. */
int hg_gumbel_halving(const hg_tree* tree, const int32_t* root_nodes, const int32_t* candidates, int C,
                      const float* base, float c_visit, float c_scale, int root_q_min_visits, int keep, int64_t B,
                      int32_t* cand_out, int64_t* chosen, void* stream);

/* ---- one simulation wave of the Gumbel root search, launched natively ----
 * The body of the reference's per-wave loop (fnn_mcts_orchestrator.py:982-1055:
 * mcts_select_replay_legal_fnn_root_slots_batch, the FNN leaf evaluation,
 * mcts_expand_and_backprop_dense_priors_batch) as one host call: select over
 * the root slots -> replay (rows of idle simulations zero) and the leaves'
 * results -> legal lists + features -> hg_fnn_leaf_eval_lists -> expansion +
 * backup (hg_mcts_expand_backprop_dense_ws), launched in that order on
 * `stream` with no host synchronisation and no allocation.  No single
 * reference entry point: it saves the host the per-call argument handling of
 * six entry points per wave.  Results are those of the six calls. */
typedef struct hg_fnn_net {   /* a 64-wide HiveFNN (fnn_network.py:97-140), F = 122 */
    const float* fc1_w;       /* [64][F] */
    const float* fc1_b;       /* [64] */
    const float* ln_w;        /* [64] */
    const float* ln_b;        /* [64] */
    const float* fc2_w;       /* [64][64] */
    const float* fc2_b;       /* [64] */
    const float* value_w;     /* [64] */
    const float* action1_w;   /* [64][128] */
    const float* action1_b;   /* [64] */
    const float* action2_w;   /* [64] */
    float value_b;
    float action2_b;
    int32_t F;
} hg_fnn_net;

typedef struct hg_wave_buffers {  /* rows for T = W * num_candidates * B simulations (or more) */
    int32_t* leaf_idx;       /* [T] */
    uint8_t* move_paths;     /* [T][128][6], each row written up to its path_lens entry */
    int32_t* path_lens;      /* [T] */
    int32_t* vl_paths;       /* [T][128], each row written up to its vl_lens entry */
    int32_t* vl_lens;        /* [T] */
    uint8_t* leaf_states;    /* [T][3424] */
    int32_t* results;        /* [T] */
    uint8_t* legal_moves;    /* [T][256][6], each row written up to its num_legal entry */
    int32_t* num_legal;      /* [T] */
    float* features;         /* [T][122], 8-byte aligned */
    float* priors;           /* [T][256], each row written up to its leaf's legal count */
    float* values;           /* [T] */
    float* child_q;          /* [T][256], each row written up to its leaf's legal count */
    void* leaf_workspace;    /* hg_fnn_leaf_eval_lists_workspace(T, 122) bytes, 256-byte aligned */
    void* tree_workspace;    /* hg_mcts_expand_backprop_dense_workspace(B, T) bytes, 4-byte aligned */
    int64_t* stats;          /* NULL, or hg_mcts_wave_stats' int64[4], accumulated */
    int64_t capacity;        /* rows each [T] array above holds */
} hg_wave_buffers;

int hg_mcts_wave_root_slots(const hg_tree* tree, const uint8_t* root_states, const int8_t* game_active,
                            const int32_t* root_nodes, const int32_t* root_slots, int num_candidates,
                            int max_root_children, float c_puct, int64_t B, int W, int deterministic_non_root,
                            float non_root_sigma, float q_penalty, const hg_fnn_net* net,
                            const hg_wave_buffers* buffers, void* stream);

/* ---- training operators ----
 * What turns a sampled batch into a step of the weights, next to the products
 * of the network's layers.  The reference trains with torch's operators
 * (hive_fnn/fnn_trainer.py, fnn_network.py:175-253); these have no entry
 * points there.  Element types of tensors: */
#define HG_F32 0
#define HG_F16 1
#define HG_BF16 2

/* Layer norm over the cols values of each row of a = x, or of a = sigmoid(x):
 * y = (a - mean) rstd weight + bias with rstd = 1 / sqrt(var + eps), var the
 * biased variance.  Row r of x begins at x + r * x_stride elements; y[rows][cols]
 * has x's type, weight / bias (NULL = 1 / 0) w_type, mean[rows] and rstd[rows]
 * are float.  rows <= 2^31 (2^21 of more than 16,384 values), cols <= 2^25. */
int hg_layer_norm_forward(const void* x, int x_type, int64_t rows, int64_t cols, int64_t x_stride,
                          const void* weight, const void* bias, int w_type, float eps, int sigmoid, void* y,
                          float* mean, float* rstd, void* stream);

/* Its gradients from dy, that of y: dx[rows][cols] in x's type, dweight[cols]
 * and dbias[cols] in w_type (each NULL = not wanted; the last two are sums over
 * all rows in one order whatever runs beside them, zeros for no rows).  mean,
 * rstd: the forward pass's.  workspace: hg_layer_norm_backward_workspace bytes,
 * 16-byte aligned, needed for dweight / dbias only. */
int64_t hg_layer_norm_backward_workspace(int64_t rows, int64_t cols);
int hg_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_type, int64_t rows, int64_t cols,
                           int64_t x_stride, const float* mean, const float* rstd, const void* weight, int w_type,
                           int sigmoid, void* dx, void* dweight, void* dbias, void* workspace, void* stream);

/* The training loss of B positions and its gradient.  Position b has n[b] =
 * num_actions[b] clamped to [0, width] legal moves; its logits are n[b] of the
 * N values of logits, the positions one after the other (the rows of
 * hg_successor_rows), its policy target the first n[b] values of row b of
 * targets[B][width] (target_type).  values[B] are the value head's results, of
 * the logits' type.
 *   losses[0] = losses[1] + value_coef * losses[2]
 *   losses[1] = sum w_b CE_b / sum w, CE_b the cross-entropy of the softmax of
 *               b's logits against its target, w = policy_weights
 *   losses[2] = sum u_b (values_b - value_targets_b)^2 / sum u, u = value_weights
 *   dlogits[N], dvalues[B] = loss_scale times the gradient of losses[0], of the
 *               logits' type
 * Positions of weight 0, without moves, or whose logits are all -inf add
 * nothing and have gradients of 0; a sum of weights of 0 counts as 1.  Logits
 * past the positions' own have gradients of 0, moves past N are left out.
 * B <= 2^26 - 4, width <= 2^31.
 * workspace: hg_policy_value_loss_workspace(B, width) bytes, 16-byte aligned. */
int64_t hg_policy_value_loss_workspace(int64_t B, int64_t width);
int hg_policy_value_loss(const void* logits, int type, int64_t N, const void* values, const int64_t* num_actions,
                         const void* targets, int target_type, int64_t width, const float* policy_weights,
                         const float* value_targets, const float* value_weights, int64_t B, float value_coef,
                         float loss_scale, float* losses, void* dlogits, void* dvalues, void* workspace,
                         void* stream);

/* One AdamW step (step >= 1) of `count` tensors, in place:
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^step) m / (sqrt(v / (1 - beta2^step)) + eps)
 * with g = grad * grad_scale[0] (NULL = 1; device memory).  `tensors` is a host
 * array, read before the call returns.  state_bits 32: exp_avg and exp_avg_sq
 * are float[count] (the scales NULL).  state_bits 8: they are float8 e4m3 codes
 * in whole blocks of HG_ADAMW_BLOCK elements, 4-byte aligned, each block with a
 * float scale: exp_avg = code * scale, exp_avg_sq = (code * scale)^2; new values
 * are rounded to a neighbouring code at random, by bits that depend on `seed`
 * and `place` + the element's index alone (place: a multiple of the block).
 * A gradient whose square passes float's range makes v inf, its weight steps by
 * 0 from then on; in 8 bits the scale of v is then inf and v of all 256 elements
 * under it inf or NaN.  An inf or NaN gradient does the same to exp_avg.
 * No tensor's param and moments may share memory with another's, nor with any
 * gradient but the param's own, element for element: the blocks that step them
 * run beside each other.
 * A tensor has under 2^34 elements (count <= 2^34 - 1024). */
#define HG_ADAMW_BLOCK 256
typedef struct hg_adamw_tensor {
    void* param;
    const void* grad;
    void* exp_avg;
    void* exp_avg_sq;
    float* exp_avg_scale;
    float* exp_avg_sq_scale;
    int64_t count;  /* elements */
    int64_t place;  /* of its first element among all states of the step */
} hg_adamw_tensor;
int hg_adamw_step(const hg_adamw_tensor* tensors, int64_t count, int param_type, int grad_type, int state_bits,
                  int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                  const float* grad_scale, uint32_t seed, void* stream);

/* ---- operators of a wider network ----
 * Its hidden block, the update of its matrices and the choice of a move from
 * its logits; no entry points of the reference.
 *
 * The gated block: gate = x Wg^T + bg, up = x Wu^T + bu, h = act(gate) up.
 * x[rows][cols] (row r at x + r * x_stride elements), w_gate and w_up
 * [hidden][cols], b_gate and b_up [hidden] (NULL = 0), and h
 * [rows][hidden] are of one type; gate and up [rows][hidden], which the backward
 * pass needs, are float, both given or both NULL (rounding them to 16 bits would
 * be a third of its results' error).  Sums are float32; float32 tensors are
 * multiplied in three bfloat16 parts a value, 24 bits (values below 2^-110 to
 * within 2^-134; an infinity times one below 2^-126 may be NaN).  rows <= 2^20, cols and
 * hidden <= 2^19, each two of them at most 2^35 together.  workspace: as many bytes, 256-byte aligned (none where that
 * is 0). */
#define HG_SIGMOID 0
#define HG_SILU 1  /* g sigmoid(g) */
#define HG_GELU 2  /* g (1 + erf(g / sqrt 2)) / 2 */
int64_t hg_gated_forward_workspace(const void* x, int type, int64_t rows, int64_t cols, int64_t x_stride,
                                   const void* w_gate, const void* w_up, int64_t hidden);
int hg_gated_forward(const void* x, int type, int64_t rows, int64_t cols, int64_t x_stride, const void* w_gate,
                     const void* w_up, int64_t hidden, const void* b_gate, const void* b_up, int act, void* h, float* gate,
                     float* up, void* workspace, void* stream);

/* Its gradients from dh[rows][hidden] (rows dh_stride elements apart), of x's
 * type, contiguous; those of the weights come together, any other is left out
 * where it is NULL.  Sums over rows are in one order whatever runs beside them.
 * The gradients of gate and up are rounded to x's type before they are
 * multiplied, which makes dx, dw_gate and dw_up of 16-bit tensors 1.35 to 1.4
 * times as far off as their own rounding does; float16's times a power of two
 * that takes the largest to 2^14 .. 2^15, so that they neither pass its 65,504
 * nor vanish, from 2^-40 of the largest up.
 * workspace: as many bytes, 256-byte aligned. */
int64_t hg_gated_backward_workspace(int type, int64_t rows, int64_t cols, int64_t hidden);
int hg_gated_backward(const void* dh, int64_t dh_stride, const void* x, int type, int64_t rows, int64_t cols,
                      int64_t x_stride, const void* w_gate, const void* w_up, int64_t hidden, const float* gate,
                      const float* up, int act, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
                      void* workspace, void* stream);

/* Which tiles these sizes take (tests and profiles ask): of h, dx, and the weights'
 * gradients, as (rows * 1000 + columns) * 100 + stages * 10 + blocks of a compute
 * unit; 0 for the kernels of narrow float32 blocks. */
int hg_gated_tiles(int type, int64_t rows, int64_t cols, int64_t hidden, int tiles[3]);

/* The Newton-Schulz iteration of `count` matrices u[rows][cols] (matrix i at
 * u + i * u_step, its row r at r * u_row elements from there):
 *   X = U / (|U| + eps), |U| the root of the sum of its squares; then `steps`
 *   times X <- a X + (b A + c A A) X, A = X X^T (X turned where it is taller than
 *   wide), (a, b, c) = coefficients[i] for step i, the last of the `triples` for
 *   the steps past them (host memory, read before the call returns)
 * out[count][rows][cols] has u's type.  Values are held in 22 bits, or to within 2^-36 of
 * |X| where that is more (so from 2^-15 of |X| down; |X| is held to its own size, however far |U| is
 * below eps): entries of X and A up to 7.9 in size, of a I + b A + c A A up to 63; past
 * that the result is inf or NaN.  rows, cols <= 2^17, count * (rows / 64 + 1)
 * (cols / 64 + 1) <= 2049^2, count <= 2^16, steps 1 to 100.
 * workspace: as many bytes, 256-byte aligned. */
int64_t hg_orthogonalize_workspace(int64_t count, int64_t rows, int64_t cols);
int hg_orthogonalize(const void* u, int type, int64_t count, int64_t rows, int64_t cols, int64_t u_row, int64_t u_step,
                     int steps, const float* coefficients, int triples, float eps, void* out, void* workspace,
                     void* stream);
/* hg_gated_tiles' numbers of A's and P's tiles, and of P X's, of up to 16 triples, 10^8
 * more where two teams of a block share a tile; 0 for matrices that a block holds. */
int hg_orthogonalize_tiles(int64_t count, int64_t rows, int64_t cols, int tiles[2]);

/* One step of `count` matrices with it, in place:
 *   m = momentum m + g;  u = g + momentum m (nesterov) or m
 *   p = p (1 - lr weight_decay) - lr scale X(u)
 * param, grad and momentum are contiguous [rows][cols]; a NULL grad leaves its
 * matrix and momentum alone.  `matrices` is a host array, read before the call
 * returns.  No param and momentum may share memory with another's, nor with any
 * gradient.  workspace: as many bytes, 256-byte aligned; two calls that are in
 * flight together must not share it. */
typedef struct hg_muon_matrix {
    void* param;
    const void* grad;
    float* momentum;
    int64_t rows, cols;
    double scale;
} hg_muon_matrix;
int64_t hg_muon_step_workspace(const hg_muon_matrix* matrices, int64_t count);
int hg_muon_step(const hg_muon_matrix* matrices, int64_t count, int param_type, int grad_type, double lr, double momentum,
                 int nesterov, double weight_decay, int steps, const float* coefficients, int triples, float eps,
                 void* workspace, void* stream);

/* A slot of each of `rows` rows of logits (row b at logits + b * stride elements),
 * drawn from uniforms[b] in [0, 1): actions[b], and with log_probs not NULL the
 * logarithm of its probability among what was kept.  Row b's slots are its first
 * num_actions[b] (NULL = width; clamped to [0, width]) without those of -inf or
 * NaN; no slot left: -1 and 0.  In order of falling logits, ties by rising slots,
 * the first top_k stay (<= 0: all), of these the fewest first ones that hold top_p
 * of their mass (>= 1: all; at least one), of these the ones at least min_p as
 * likely as the first.  The slot drawn is the first, in the slots' order, at which
 * the running sum of the weights kept, exp((x - max) / T), passes u times their
 * whole.  T not above 0: the largest logit's first slot, of probability 1.
 * Each setting is an array of a value a row, or where that is NULL the number
 * beside it.  NaN: a temperature takes the largest, top_p and min_p leave all, a
 * uniform number is 0.  width <= 2^20, rows <= 2^25 (2^21 of more
 * than 1,024 slots). */
int hg_sample_actions(const void* logits, int type, int64_t rows, int64_t width, int64_t stride,
                      const int64_t* num_actions, const float* uniforms, const float* temperatures, double temperature,
                      const int64_t* top_ks, int64_t top_k, const float* top_ps, double top_p, const float* min_ps,
                      double min_p, int64_t* actions, float* log_probs, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HIVE_GPU_H */
