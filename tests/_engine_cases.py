"""Sizes of the projection (tokens, in_features, out_features) and of the feed-forward block (tokens, hidden, inner,
out_features) that together reach every engine, tile and way of splitting K in each of their products, off the tiles'
borders.  tests/test_layer_plans.py holds that they do."""
from __future__ import annotations

LINEAR16 = [
    (17, 26, 26), (17, 5891, 6271), (3808, 70, 5369), (4589, 4957, 65), (1989, 1566, 692), (67, 6186, 5659), (2953, 65, 8539),
    (2263, 6329, 1929), (4271, 1578, 2938), (4941, 966, 5756),
]
LINEAR32 = [(17, 28, 25), (284, 610, 205), (3541, 2246, 65), (65, 6173, 733), (1318, 33, 4771)]
BLOCK16 = [
    (17, 32, 25, 26), (1322, 35, 1747, 40), (18, 4881, 3976, 2039), (4890, 4667, 74, 4294), (1882, 675, 822, 2156),
    (4150, 67, 3576, 38), (197, 51, 4098, 3442), (4724, 81, 719, 1347), (1298, 3856, 298, 139), (1432, 1454, 4109, 113),
    (4182, 3017, 701, 589), (574, 51, 3625, 1812), (5920, 36, 2126, 2213), (1374, 3196, 4183, 607), (1323, 43, 4123, 3018),
    (1373, 1201, 3174, 4985), (3919, 2856, 1509, 27),
    (4135, 3840, 512, 563), (656, 640, 3840, 6460),  # the ring engine's K ranges of K-major operands: K a multiple of 64
    (48, 4096, 1100, 520),                           # a decoding batch
]
BLOCK32 = [(18, 39, 26, 27), (2441, 34, 1325, 44), (73, 3536, 852, 395), (1549, 2565, 204, 2245), (232, 45, 718, 4176)]

TILES16 = [("tile", 64, 64), ("tile", 64, 128), ("tile", 128, 128), ("ring", 256, 256)]
TILES32 = [("split3", 64, 64), ("split3", 256, 128)]


def reached(plans):
    """{(product, engine, tile rows, tile columns, K in ranges)} over a list of plans."""
    return {(name, p["engine"], p["tile_rows"], p["tile_cols"], p["splits"] > 1) for plan in plans for name, p in plan.items()}


def every(products, tiles):
    return {(name, *t, split) for name in products for t in tiles for split in (False, True)}
