"""Sizes that take every kernel of the MX products, over several of its steps, with odd rows
and columns: (form, act, rows, K, N, activations of 16 bits)."""

BOTH = ("fp8", "fp4")
CASES = [
    # streamed: row tiles of the weight, of the activations, quantized in place, K shared
    *[(form, act, M, K, n, x) for act in BOTH for form, n in (("plain", 97), ("gated", 83), ("gated mx", 96)) for M, K, x in
      ((3, 544, True), (5, 2080, True), (2, 4128, True), (7, 544, False), (16, 4128, False), (19, 544, False), (29, 4128, True))],
    *[(form, act, M, K, n, x) for act in BOTH for form, n in (("plain", 97), ("gated", 83)) for M, K, x in
      ((37, 544, False), (47, 4128, True), (51, 544, True), (64, 4128, False))],
    *[("plain", act, M, K, N, x) for act in BOTH for M, K, N, x in
      ((13, 1056, 20001, False), (11, 6176, 2500, False), (17, 1056, 11003, True), (31, 6176, 2500, True), (33, 1568, 8209, False),
       (41, 6176, 2500, True), (50, 2080, 6600, True), (55, 6176, 2500, False), (21, 2592, 11003, True))],
    ("plain", "fp4", 45, 6176, 5003, True),
    *[("gated", act, M, K, N, True) for act in BOTH for M, K, N in ((18, 1568, 8209), (27, 2080, 7003))],
    ("gated", "fp4", 40, 6176, 2500, False),
    # by tiles: few rows by wide weights, then small, middle and large tiles, with more stages or fewer
    *[(form, act, M, K, N, x) for act in BOTH for form, N in (("plain", 13001), ("gated", 11003), ("gated mx", 11008)) for M, K, x in
      ((33, 1568, True), (61, 2080, False))],
    *[("plain", act, 26, 1568, 16395, True) for act in BOTH], *[("gated", act, 30, 1568, 11003, False) for act in BOTH],
    *[("gated mx", act, 31, 6176, 11008, True) for act in BOTH],
    *[(form, act, 200, 1824, N, True) for act in BOTH for form, N in (("plain", 515), ("gated", 259), ("gated mx", 288))],
    *[(form, "fp4", 1900, 1568, N, True) for form, N in (("plain", 4001), ("gated", 2001), ("gated mx", 2016))],
    *[(form, "fp4", 1900, 1568, N, True) for form, N in (("plain", 8001), ("gated", 4001), ("gated mx", 4064))],
    ("plain", "fp8", 1000, 1568, 6101, True), ("plain", "fp8", 1900, 8224, 4100, True),
    *[(form, "fp8", 1900, 1568, N, False) for form, N in (("plain", 4100), ("gated", 2113), ("gated mx", 2144))],
]
