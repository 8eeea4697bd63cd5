"""ngram_amd: an MI355X-native engine for the n-gram hint path of hermabr/n-gram-hinted-lm.

Host code (Python on PyTorch-ROCm) over a C-ABI HIP library (csrc/, built for gfx950 by ngram_amd.build). Modules:
  data            shard files and the seeded synthetic streams of the benchmark configurations
  lib             the ctypes binding (the reference's Lib convention)
  gpu_val_stats   the validation-side statistics driver (old_records/gpu_val_stats.py on one GPU)
  count_table     corpus-wide exact count tables on the GPU (exact_match CountTable's surface) + hint queries
  hints           the hint directory's writer and reader, HintRows
  embed           hint rows and tokens embedded, with the table's and the weights' gradients (HintEmbedding)
  kvcache         a paged key/value cache in 8 or 16 bits, quantised as it is written
  tree            attention for trees of drafted tokens over that cache
  beam            a beam search's step over a model's logits, and its states' reordering
  pages           who holds that cache's pages: forks, room for more tokens, copies, moves
  sparse          attention over the pages that a cheap score keeps for each token
"""
__all__ = ["data", "lib", "build"]
