#!/usr/bin/env python3
"""
Scores texts with a decoder-only language model and continues them, over a paged key / value cache (returnn_b200/models/paged_decoder.py).
The model is a small one with random parameters; load a checkpoint into it, or import one (returnn_b200/frontend/conversions/hf_llama.py).
"""

import argparse

import _setup_env  # noqa
import torch
import returnn_b200.frontend as rf
from returnn_b200.tensor import Dim
from returnn_b200.frontend.decoder.transformer import TransformerDecoder, FeedForwardGated
from returnn_b200.models.paged_decoder import PagedDecoder


def main():
    """main"""
    arg_parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    arg_parser.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    arg_parser.add_argument("--layers", type=int, default=2)
    arg_parser.add_argument("--requests", type=int, default=4)
    arg_parser.add_argument("--max-new", type=int, default=8)
    args = arg_parser.parse_args()
    rf.select_backend_torch()
    torch.manual_seed(42)
    model = TransformerDecoder(
        None, Dim(1000, name="vocab"), Dim(512, name="model"), num_layers=args.layers, num_heads=8, pos_enc=None, norm=rf.build_dict(rf.RMSNorm),
        ff=rf.build_dict(FeedForwardGated), dropout=0.0, att_dropout=0.0, share_embedding=False, input_embedding_scale=1.0,
        layer_opts=dict(self_att=rf.build_dict(rf.RotaryPosCausalSelfAttention, with_bias=False, qk_norm=True)))
    for param in model.parameters():
        value = param.raw_tensor.detach()
        if value.dim() > 1:
            value = torch.randn(value.shape) * value.shape[0] ** -0.5
        param.raw_tensor = torch.nn.Parameter(value.to(args.device), requires_grad=False)
    paged = PagedDecoder(model, max_requests=args.requests, max_len=64, dtype=torch.bfloat16 if args.device == "cuda" else None)
    texts = [torch.randint(1, 1000, (n,)).tolist() for n in (5, 30, 12, 17, 3, 44)]  # more than run at a time
    for text, scores in zip(texts, paged.score(texts, num_top=3)):
        print("text of %2i labels: log probability %8.2f, entropy %.2f per label, best after the first: %s" % (
            len(text), float(scores.log_probs.sum()), float(scores.entropy.mean()), scores.top_labels[0].tolist()))
    for text, more in zip(texts, paged.generate(texts, max_new=args.max_new, eos=0)):
        print("after %2i labels: %s (log probability %.2f)" % (len(text), more.labels, sum(more.log_probs)))


if __name__ == "__main__":
    main()
