#pragma once
// Layers, loss and optimiser on top of Tensor.  The first part mirrors the
// reference's include/micrograd/nn.h:6-34; the marked additions are what batched
// softmax-cross-entropy training and inference on the GPU need.

#include <memory>
#include <string>
#include <vector>

#include "Tensor.h"
#include "detail/GradBuckets.h"

std::shared_ptr<Tensor> mse_loss(const std::shared_ptr<Tensor> &prediction,
                                 const std::shared_ptr<Tensor> &target);
std::shared_ptr<Tensor> avg_pool_2x2(const std::shared_ptr<Tensor> &input);

class Linear {
public:
  Linear(size_t in_features, size_t out_features);
  // input [B, in] -> [B, out] for any batch size B: one GEMM with the bias add
  // fused into its epilogue.
  std::shared_ptr<Tensor> forward(const std::shared_ptr<Tensor> &input);
  std::shared_ptr<Tensor> weights();
  std::shared_ptr<Tensor> bias();

  // addition: relu(forward(input)) as a single node (bias + ReLU epilogue).
  // When the node feeding gradient into it is another Linear, that layer's dX
  // GEMM applies this node's ReLU mask in its epilogue; grad() of the returned
  // tensor then holds the gradient with respect to the pre-activation.
  std::shared_ptr<Tensor> forward_relu(const std::shared_ptr<Tensor> &input);

private:
  std::shared_ptr<Tensor> fused_forward(const std::shared_ptr<Tensor> &input, bool relu);
  std::shared_ptr<Tensor> weights_;
  std::shared_ptr<Tensor> bias_;
};

namespace micrograd {
enum class Activation { None, ReLU, SiLU };  // SiLU: z / (1 + exp(-z))
}

// addition: group norm with an activation, channels last.  forward([N, ..., channels])
// normalises, for each of the N samples, the values of every group of channels /
// groups neighbouring channels over all positions between (none for [N, channels]) to
// mean 0 and variance 1 / (1 + eps / variance), scales and shifts each channel by
// weights() (1 at first) and bias() (0), and applies the activation, as one node.
class GroupNorm {
public:
  GroupNorm(size_t groups, size_t channels, double eps = 1e-5);
  std::shared_ptr<Tensor> forward(const std::shared_ptr<Tensor> &input,
                                  micrograd::Activation activation = micrograd::Activation::None);
  std::shared_ptr<Tensor> weights();
  std::shared_ptr<Tensor> bias();

private:
  size_t groups_, channels_;
  double eps_;
  std::shared_ptr<Tensor> weights_;
  std::shared_ptr<Tensor> bias_;
};

class SGD {
public:
  SGD(std::vector<std::shared_ptr<Tensor>> parameters, double learning_rate);
  ~SGD();

  void step();
  void zero_grad();

  // addition: moves all parameters and their gradients into two flat device
  // buffers and, when a communicator is up (micrograd::comm_init), sums each
  // parameter's gradient across ranks as soon as backward() has finished it.
  // step() then waits for those sums on the device, not on the host.
  // Parameters travel in one message per layer: a weight directly followed by
  // its bias forms a pair, anything else goes alone.  A parameter that the
  // backward sweep never reaches is reduced by step() itself, and a second
  // backward() before step() throws std::logic_error once sums have been
  // exchanged (they cannot be accumulated into).
  void enable_allreduce();

private:
  void on_grad_ready(size_t index);
  std::vector<std::shared_ptr<Tensor>> parameters_;
  double learning_rate_;
  // flat storage (after enable_allreduce)
  double *flat_data_ = nullptr;
  double *flat_grad_ = nullptr;
  std::vector<size_t> offsets_;
  micrograd::detail::GradBuckets buckets_;
  void reduce_bucket(size_t bucket);
  std::vector<char> requires_flags() const;
  size_t flat_elems_ = 0;
  bool allreduce_ = false;
};

void save_model(const std::string &path, Linear &l1, Linear &l2);
void load_model(const std::string &path, Linear &l1, Linear &l2);

// ---- additions ------------------------------------------------------------
// Mean softmax cross-entropy of logits [B, C] against class ids.  `labels` is a
// tensor of B class ids stored as doubles (shape [B] or [B,1]) or a host vector.
// `denom` overrides the divisor of the mean (0 = B); a rank holding a shard of a
// global batch passes the global batch size.
std::shared_ptr<Tensor> softmax_cross_entropy(const std::shared_ptr<Tensor> &logits,
                                              const std::shared_ptr<Tensor> &labels,
                                              double denom = 0.0);
std::shared_ptr<Tensor> softmax_cross_entropy(const std::shared_ptr<Tensor> &logits,
                                              const std::vector<int> &labels, double denom = 0.0);
// The same loss of head.forward(input) for heads with many classes, without the [B, C]
// logits: they exist for a block of rows at a time (at most 1 GiB).  The gradients are
// computed in the forward pass, which has the block's logits at hand (three products
// instead of the four that going through them again in the backward pass would take),
// and kept for backward(), which scales them by its own gradient, in buffers of the size
// of what they belong to, until the graph goes; where neither the input nor the head's parameters require a
// gradient only the loss is computed (backward() throws std::logic_error for one that
// came to require a gradient later).  A row with label -1 is left out (a padded
// batch): it adds nothing to the loss or any gradient, whatever its values are; it does
// count in the default divisor.
std::shared_ptr<Tensor> linear_cross_entropy(const std::shared_ptr<Tensor> &input, Linear &head,
                                             const std::shared_ptr<Tensor> &labels, double denom = 0.0);
std::shared_ptr<Tensor> linear_cross_entropy(const std::shared_ptr<Tensor> &input, Linear &head,
                                             const std::vector<int> &labels, double denom = 0.0);
// Index of the first strict maximum of each row of a 2-D tensor.
std::vector<int> argmax_rows(const std::shared_ptr<Tensor> &x);
