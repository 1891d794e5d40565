"""Sizes of the paged attention's sharper tests, shared by the tests on the CPU and on the GPU."""
from paged_bounds import BF16, F16

# a query's low bits: few rows (mma.sync) and many (tcgen05), every padded width
SPLIT = [dict(dtype=dt, D=D, T=T, P=16) for dt in (F16, BF16) for D in (32, 64, 96, 128) for T in (8, 80)] + [
    dict(dtype=BF16, D=D, T=T, P=64) for D in (160, 256) for T in (8, 40)]

# single slots: one sequence (cluster form, long lists), batches, windows, pages that end inside a tile
TELLING = [
    dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=64, lens=[700, 64, 1, 63, 65]),
    dict(dtype=BF16, H=32, Hkv=8, T=1, D=128, P=16, lens=[4096]),
    dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=64, lens=[20011]),
    dict(dtype=F16, H=4, Hkv=4, T=1, D=64, P=100, lens=[1500, 333]),
    dict(dtype=BF16, H=2, Hkv=1, T=3, D=256, P=72, lens=[900, 5]),
    dict(dtype=F16, H=4, Hkv=2, T=16, D=256, P=16, lens=[600, 129]),
    dict(dtype=F16, H=8, Hkv=2, T=8, D=96, P=8, lens=[500, 40], kind="tree"),
    dict(dtype=F16, H=8, Hkv=2, T=40, D=128, P=16, lens=[1000, 63, 0]),
    dict(dtype=BF16, H=8, Hkv=2, T=64, D=128, P=72, lens=[3000, 65], kind="tree"),
    dict(dtype=F16, H=6, Hkv=2, T=130, D=64, P=64, lens=[900, 128], kind="tree"),
    dict(dtype=BF16, H=4, Hkv=1, T=300, D=128, P=100, lens=[450]),
    dict(dtype=F16, H=8, Hkv=2, T=1, D=128, P=16, lens=[900, 100], window=130),
    dict(dtype=F16, H=4, Hkv=2, T=30, D=128, P=16, lens=[900, 100], window=130),
]

# rising maxima: segments of one tile (few units), of several (single sequences, batches), split over CTAs
RISING = [
    *[dict(dtype=dt, H=4, Hkv=2, T=32, D=D, P=64, lens=[600], pattern=pat, step=10)
      for dt in (F16, BF16) for D in (64, 128) for pat in ("every", "second", "end")],
    *[dict(dtype=dt, H=16, Hkv=8, T=64, D=128, P=16, lens=[1000, 900, 1000, 333], pattern=pat, step=step, rows=rows)
      for dt, pat, step, rows in ((F16, "every", 10, "odd"), (BF16, "every", 10, "warps"), (BF16, "second", 20, "odd"),
                                  (F16, "second", 7, "all"), (BF16, "end", 10, "warps"))],
    dict(dtype=BF16, H=16, Hkv=8, T=40, D=64, P=64, lens=[64 * k for k in (1, 2, 3, 5, 8, 13, 20, 21, 20, 13, 8, 5)],
         pattern="every", step=10, rows="odd"),
    dict(dtype=BF16, H=16, Hkv=8, T=40, D=128, P=64, lens=[64 * k for k in (1, 2, 3, 5, 8, 13, 20, 21, 20, 13, 8, 5)],
         pattern="every", step=10, rope=True),
    dict(dtype=F16, H=8, Hkv=1, T=64, D=128, P=100, lens=[500], pattern="every", step=10, rows="odd"),
    # few rows: the same on mma.sync, where every growth rescales
    dict(dtype=BF16, H=16, Hkv=4, T=1, D=128, P=64, lens=[700, 1400], pattern="every", step=10, rows="odd"),
    dict(dtype=BF16, H=4, Hkv=2, T=12, D=256, P=64, lens=[700, 200], pattern="every", step=10, rows="odd"),
]

# several units to a CTA: one and two row tiles, fewer and more than 32 list entries, one-tile units
MANY_UNITS = [
    dict(dtype=F16, H=16, Hkv=8, T=40, D=128, P=64, lens=[(i * 37) % 400 for i in range(40)], kind="tree", window=-1),
    dict(dtype=BF16, H=16, Hkv=8, T=80, D=128, P=16, lens=[(i * 53) % 400 for i in range(24)], kind="tree", window=-1),
    dict(dtype=F16, H=8, Hkv=8, T=20, D=64, P=64, lens=[i % 40 for i in range(70)], kind="chain", window=-1),
    dict(dtype=BF16, H=20, Hkv=10, T=33, D=64, P=72, lens=[(i * 71) % 600 for i in range(30)], kind="tree", window=90),
    dict(dtype=F16, H=32, Hkv=16, T=100, D=96, P=16, lens=[0, 300, 150, 64, 1, 800, 77, 20, 500, 450, 333], kind="chain",
         window=-1),
    dict(dtype=F16, H=8, Hkv=8, T=3, D=128, P=16, lens=[(i * 29) % 300 for i in range(60)], kind="tree", window=50),
]
