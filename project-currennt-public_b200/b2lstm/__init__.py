"""b2lstm: Python harness over libb2lstm.so, the B200 implementation of the CURRENNT peephole
LSTM / BLSTM training path.  The library is the product; this package only loads it (ctypes),
generates the synthetic workloads and launches processes.  There is no CPU fallback: importing
works without a GPU (symbols can be inspected), every compute call needs one.
"""
from .lib import (B2Error, LstmLayer, Net, lib, library_path, lstm_num_weights, matrix_multiply, matrix_multiply_noalloc,
                  dp_unique_id, DataSet, data_reseed, train_epoch, train_epoch_batch, write_nc, Optimizer)
from .operators import (StateList, TensorList, beam_reorder, beam_select, beam_select_workspace, block_norm_backward, block_norm_backward_workspace, block_norm_forward, distill_backward,
                        distill_forward, embedding_backward, embedding_backward_workspace, embedding_forward, gradient_clip, gradient_norm, gradient_norm_workspace,
                        int8_product, int8_product_workspace, int8_quantize, logprob_backward, logprob_forward)
from . import workloads

__all__ = ["B2Error", "LstmLayer", "Net", "lib", "library_path", "lstm_num_weights", "matrix_multiply", "matrix_multiply_noalloc",
           "dp_unique_id", "DataSet", "data_reseed", "train_epoch", "train_epoch_batch", "write_nc", "Optimizer", "workloads", "TensorList", "block_norm_backward", "block_norm_backward_workspace",
           "block_norm_forward", "embedding_backward", "embedding_backward_workspace", "embedding_forward", "gradient_clip", "gradient_norm",
           "gradient_norm_workspace", "logprob_backward", "logprob_forward", "StateList", "beam_reorder", "beam_select", "beam_select_workspace", "distill_backward",
           "distill_forward", "int8_product", "int8_product_workspace", "int8_quantize"]
