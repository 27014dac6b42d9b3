"""Products that between them take every form of th_gemm_i8 on a card of 256 CUs, with remainders in rows, channels and k:
(form, m, k, n).  test_i8_host.py asks the rule for each; test_gpu_i8_forms.py runs them."""
FORMS = ["rows 1x1", "rows 1x2", "rows 2x2", "rows 1x4", "rows 2x4", "rows 3x4", "tile 64x64", "tile 64x128, two groups", "tile 64x128", "tile 128x128",
         "tile 128x256", "tile 256x256"]
SIZES = [
    ("rows 1x1", 16, 2047, 4107), ("rows 1x1", 5, 577, 12300),
    ("rows 1x2", 17, 1090, 4090), ("rows 1x2", 32, 1, 15), ("rows 1x2", 31, 4160, 2001),
    ("rows 2x2", 17, 999, 4113), ("rows 2x2", 31, 65, 8203), ("rows 2x2", 32, 2112, 12289),
    ("rows 1x4", 33, 500, 4096), ("rows 1x4", 61, 2049, 333), ("rows 1x4", 64, 640, 1000),
    ("rows 2x4", 33, 1000, 4107), ("rows 2x4", 61, 2111, 8190), ("rows 2x4", 64, 64, 4500),
    ("rows 3x4", 33, 1501, 12307), ("rows 3x4", 61, 4096, 11008), ("rows 3x4", 64, 333, 8201), ("rows 3x4", 49, 63, 16400),
    ("tile 64x64", 65, 700, 17), ("tile 64x64", 131, 4097, 500), ("tile 64x64", 201, 64, 1003),
    ("tile 64x128, two groups", 72, 613, 8295), ("tile 64x128, two groups", 67, 140, 8473), ("tile 64x128, two groups", 100, 2300, 11007),
    ("tile 64x128", 394, 616, 8298), ("tile 64x128", 388, 72, 8277), ("tile 64x128", 385, 1089, 8257),
    ("tile 128x128", 321, 626, 5499), ("tile 128x128", 532, 3, 5565), ("tile 128x128", 509, 2047, 5631),
    ("tile 128x256", 527, 612, 7239), ("tile 128x256", 707, 68, 6875), ("tile 128x256", 1030, 1220, 4097),
    ("tile 256x256", 2750, 601, 4363), ("tile 256x256", 1537, 201, 7589), ("tile 256x256", 2051, 1030, 6001),
]
