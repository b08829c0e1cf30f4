"""Shapes of the tree attention at which blocks of 64 query rows meet wide heads:
(contexts, nodes of each tree, heads, KV heads, head_dim, window)."""
WIDE = {
    "full_layer": ([9000], [64], 8, 2, 512, 0),             # eight chunks of dims, four dim blocks
    "three_ring_slots": ([12000], [40], 8, 2, 512, 0),      # the last row block 32 rows short
    "window_inside_tiles": ([9000], [64], 8, 2, 512, 8500),
    "half_the_dims": ([6000], [40], 8, 2, 256, 0),
    "unaligned_rows": ([7001], [33], 8, 2, 450, 0),         # rows on 8-byte boundaries, the last chunk two dims
    "short_last_chunk": ([10007], [64], 8, 1, 388, 0),      # eight heads of one KV head, four dims in the last block
    "ragged_batch": ([128, 4097, 1639, 3150, 692, 2203, 3714, 1256, 2767, 309, 1820, 3331, 873, 2384, 1, 0],
                     [11, 9, 13, 1, 11, 24, 3, 11, 7, 16, 11, 2, 11, 20, 11, 5], 8, 2, 512, 0),
}
