"""Products of 8-bit rows that take each form (fastertnn_amd/csrc/i8_forms.h): tokens, channels and lengths of rows."""

# form: (m, n), and the lengths: none of a step's 128 codes, one step, steps and a part, more steps than a ring holds
TILES = {
    "T256": ((4096, 3999), (40, 128, 700)),
    "T128": ((1000, 4001), (16, 128, 257, 1168)),
    "T128Two": ((2000, 3990), (100, 256, 900)),
    "T128x64": ((500, 3999), (16, 384, 1000)),
    "T64": ((200, 2999), (17, 128, 512, 1168, 2052)),
    "T64Split": ((130, 1500), (8192, 9000, 8336)),
}
# (nb, mb): (m, n) for codes and for packed rows
FEW_CODES = {(1, 1): (33, 1000), (1, 2): (50, 2001), (2, 1): (9, 8001)}
FEW_PACKED = {(1, 1): (33, 1000), (2, 1): (20, 4500), (4, 1): (15, 21001), (4, 2): (32, 11003), (4, 4): (200, 4003)}
FEW_K = (16, 1025, 5000)   # lengths of a row at which the packed ones have their form
TILES_PACKED = ("T256", "T128Two")   # those of the above whose longest rows run as tiles when packed
