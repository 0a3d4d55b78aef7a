"""The guide's example of a serving program, as text: a GPU test runs it, and a CPU
test holds the guide to it."""

SETUP = '''
table = rt.rope_table(128, 10000.0, scaling="turns", factor=8, trained=8192, fast=4, slow=1)  # once
cache = rt.KvCache.empty(pages, 8, 64, 128, torch.float8_e4m3fn, block_table=block_table)     # once
# (In 8 bits with a scale for 32 slots: KvCache.empty(..., torch.int8, block_table=..., scale_block=32).)
'''

STEP = '''
# A prompt, or a chunk of one: keys ctx .. ctx + new - 1 of each sequence.
rt.rope(q, q, None, table, k=k, k_out=k, start=ctx)
rt.kv_append(k, v, cache, ctx, new_len=new)       # new: tokens of each sequence
rt.tree_attn(q, cache, ctx, o, new_len=new)       # token t sees ctx and the new ones up to itself
ctx += new

# A step of drafted trees: node 0 is the last token that is decided, parents[b, t] the node that
# draft t continues (-1: the context), nodes[b] their number (0: sequence b has ended).
mask, depth = rt.tree_mask(parents)               # once a step, for all layers
rt.rope(q, q, depth, table, k=k, k_out=k, start=ctx)
rt.kv_append(k, v, cache, ctx)
rt.tree_attn(q, cache, ctx, o, mask=mask)
# uniform [batch, tokens] and final [batch]: the step's random numbers.
path, count, token = rt.tree_verify(logits, drafts, parents, uniform, final, temperature=temperature,
                                    new_len=nodes)
if cache.scale_block == 1:                        # every layer: the accepted branch moves to its place
    rt.kv_compact(cache, path, ctx, count)
else:                                             # rows that share scales do not move: appended again
    at = path.clamp(min=0).long()[:, None, :, None].expand(k.shape)
    rt.kv_append(k.gather(2, at), v.gather(2, at), cache, ctx, new_len=count)
ctx += count                                      # `token` is the next tree's node 0
'''

FORK = '''
# Sequence b goes on as sequence parent[b] (beams, several answers to a prompt), or ends: parent[b] = -1.
# It takes over the parent's length, which kv_pages takes, its next root and its nodes.
up, ends = parent.clamp(min=0).long(), parent < 0
ctx, token, nodes = torch.where(ends, -1, ctx[up]), token[up], torch.where(ends, 0, nodes[up])
moved, src, dst, rows, lacking = rt.kv_pages(block_table, ctx, ctx + tokens, 64, pages, parent=parent)
block_table.copy_(moved)                          # sequences share their whole pages
rt.kv_copy_pages(cache, src, dst, rows=rows)      # every layer: what they write on is their own
'''

REST = '''
# Images and video: positions [axes, batch, tokens] in time, height and width.
axis = rt.rope_axes([16, 24, 24])                 # once: the axis of each pair
rt.rope(q, q, positions, table, k=k, k_out=k, pair_axis=axis)
rt.rope(dy, dx, positions, table, pair_axis=axis, backward=True)  # the gradient

rt.kv_read(cache, k16, v16, start)                # keys start .. of each sequence, as bf16 / f16
'''
