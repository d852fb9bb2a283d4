"""Shapes of attention that reach rare states of its kernels, and the arithmetic that shows that they do."""

# (B, T, H, Hk, D), in order and 16-bit: parts of dk and dv without a tile of queries, beside full blocks of keys
PARTS_WITHOUT_TILES = [(1, 1024, 8, 4, 128), (1, 1024, 8, 4, 96), (2, 1024, 8, 8, 128), (1, 384, 4, 1, 128), (2, 1000, 8, 4, 96)]


def dkv_parts(B, Tq, Tk, H, Hk, D, causal):
    """Parts that the sums of dk and dv of a 16-bit call are split into (plan_of in csrc/wst_attention.hip)."""
    group, keys = H // Hk, B * Hk * -(-Tk // 128)
    items = group * -(-Tq // 64)
    want = 1024 if causal and D <= 64 else 512
    parts = min(max(min(-(-want // keys), items // 2), 1), 64)
    even = parts
    while even % group and group % even:
        even += 1
    return even if even < 2 * parts else parts


def parts_without_tiles(B, T, H, Hk, D):
    """(sequence and key head, block of 128 keys, part) of a call in order that has keys to spare in the block's second
    half and no tile of queries to walk: k_attn_dkv's division of tiles among parts (csrc/wst_attention.h)."""
    group, parts, found = H // Hk, dkv_parts(B, T, T, H, Hk, D, True), []
    for j0 in range(0, T, 128):
        tiles = -(-T // 64) - j0 // 64                      # tiles of 64 queries that see a key of the block
        for part in range(parts):
            if parts % group == 0:
                without = part // group >= tiles            # one head a part, every parts / group-th of its tiles
            elif group % parts == 0:
                without = tiles == 0
            else:
                without = part >= group * tiles
            if without and T - j0 > 64:
                found += [(cell, j0, part) for cell in range(B * Hk)]
    return found
