"""Sizes of the 8-bit product that reach each of its kernels: (kernel of the rule, rows 16-byte aligned) -> (m, n) and k.

m and n are no multiples of the tiles; k ends in front of, at and behind a stage of 128 and a unit of 16, with none, one and several whole
stages in front."""
DEPTHS = (64, 127, 128, 129, 143, 145, 255, 256, 1025)
SHAPES = {
    ("kLinear256", True): (((2305, 3841), (4100, 2050)), DEPTHS),
    ("kLinear128", True): (((1500, 4100), (3000, 2050)), DEPTHS),
    ("kLinear64Deep", True): (((520, 520), (100, 3000)), (1000, 1023, 1024, 1025, 1279, 1280, 1295, 1297, 1407)),
    ("kLinear64", True): (((1030, 3000), (700, 4100)), (33,) + DEPTHS),
    ("kLinearFew", True): (((1, 1000), (17, 70), (100, 300)), (33, 15) + DEPTHS),
    ("kLinear128", False): (((700, 3001), (1030, 2050)), (33,) + DEPTHS),
    ("kLinearFew", False): (((1, 1000), (17, 70), (100, 300)), (33, 15) + DEPTHS),
}
CASES = [(kernel, whole, m, n, k) for (kernel, whole), (sizes, depths) in SHAPES.items() for m, n in sizes for k in depths]
